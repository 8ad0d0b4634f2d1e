// Low-rank adapters of many requests beside a shared projection, and their
// gradients.  Row r is (token t, slot i); its adapter is adapters[t] (-1: none)
// and its expert ids[t][i] (0 without ids); A and B are the pair of that key.
//   forward    s = A x_r;  y_r = base_r + scale B s
//   backward   u = scale B^T dy_r;  dx_r (+)= A^T u;  dA (+)= u x_r^T;  dB (+)= scale dy_r s^T
// Sums are f32; weights of f16 and bf16 are widened exactly.
#pragma once
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

namespace sabah {

constexpr int kLoraThreads = 256;
constexpr int kLoraMaxRank = 128;
constexpr unsigned kErrLora = 4u;             // sticky error word: an adapter or expert id out of range
constexpr int kLoraNone = -1, kLoraBad = -2;  // keys of a row without an adapter, and of one with a bad id

struct LoraArgs {
    const uint8_t* x;             // row (t, i): x + t * x_tok + (i % x_rows) * x_id
    size_t x_id, x_tok;
    const int32_t* adapters;      // [n_tokens]
    const uint8_t* ids;           // int32, or null
    size_t ids_id, ids_tok;
    int x_rows, n_ids, n_tokens;
    const void *a, *b;            // [n_adapters][n_experts][rank][k], [n_adapters][n_experts][rows][rank]
    const float* scale;           // [n_adapters], or null
    const int32_t* ranks;         // [n_adapters], or null
    int n_adapters, n_experts, rank, k, rows;
    const uint8_t* base;          // forward: or null
    size_t base_id, base_tok;
    uint8_t* dst;
    size_t dst_id, dst_tok;
    // backward
    const uint8_t* dy;
    size_t dy_id, dy_tok;
    uint8_t* dx;                  // or null
    size_t dx_id, dx_tok;
    float *da, *db;               // or null
    int add_dx, add_dw;
    float* su;                    // [rows of the call][2 rank]: s, u
    unsigned int* err;
};

typedef float lf4 __attribute__((ext_vector_type(4)));
typedef uint16_t lu4 __attribute__((ext_vector_type(4)));
typedef uint16_t lu8 __attribute__((ext_vector_type(8)));
// the same at any address of the element's alignment (one load all the same)
typedef lf4 lf4u __attribute__((aligned(4)));
typedef lu4 lu4u __attribute__((aligned(2)));
typedef lu8 lu8u __attribute__((aligned(2)));

// Storage types: four and eight neighbours as loaded, and a value of them in f32
struct LoraF32 {
    typedef float T;
    struct V4 { lf4 v; };
    struct V8 { lf4 v[2]; };
    static __device__ inline V4 load4(const T* p) { return {*reinterpret_cast<const lf4u*>(p)}; }
    static __device__ inline V8 load8(const T* p) {
        return {{*reinterpret_cast<const lf4u*>(p), *reinterpret_cast<const lf4u*>(p + 4)}};
    }
    static __device__ inline float value(T w) { return w; }
    static __device__ inline float get(const V4& v, int c) { return v.v[c]; }
    static __device__ inline float get(const V8& v, int c) { return v.v[c >> 2][c & 3]; }
    static __device__ inline void set(V4& v, int c, T w) { v.v[c] = w; }
    static __device__ inline void set(V8& v, int c, T w) { v.v[c >> 2][c & 3] = w; }
};
template <typename W>
struct Lora16 {
    typedef uint16_t T;
    struct V4 { lu4 v; };
    struct V8 { lu8 v; };
    static __device__ inline V4 load4(const T* p) { return {*reinterpret_cast<const lu4u*>(p)}; }
    static __device__ inline V8 load8(const T* p) { return {*reinterpret_cast<const lu8u*>(p)}; }
    static __device__ inline float get(const V4& v, int c) { return W::value(v.v[c]); }
    static __device__ inline float get(const V8& v, int c) { return W::value(v.v[c]); }
    static __device__ inline void set(V4& v, int c, T w) { v.v[c] = w; }
    static __device__ inline void set(V8& v, int c, T w) { v.v[c] = w; }
};
struct LoraF16 : Lora16<LoraF16> {
    static __device__ inline float value(T w) { return __half2float(__ushort_as_half(w)); }
};
struct LoraBF16 : Lora16<LoraBF16> {
    static __device__ inline float value(T w) { return __uint_as_float((uint32_t)w << 16); }
};

// the row's key: adapter * n_experts + expert, kLoraNone or kLoraBad
__device__ inline int lora_key(const LoraArgs& a, int row) {
    const int t = row / a.n_ids, i = row - t * a.n_ids, ad = a.adapters[t];
    if (ad == -1) return kLoraNone;
    const int e = a.ids ? *reinterpret_cast<const int32_t*>(a.ids + (size_t)t * a.ids_tok + (size_t)i * a.ids_id) : 0;
    if (ad < 0 || ad >= a.n_adapters || e < 0 || e >= a.n_experts) return kLoraBad;
    return ad * a.n_experts + e;
}
__device__ inline int lora_rank(const LoraArgs& a, int key) {
    return a.ranks ? max(0, min(a.rank, a.ranks[key / a.n_experts])) : a.rank;
}
__device__ inline float lora_scale(const LoraArgs& a, int key) { return a.scale ? a.scale[key / a.n_experts] : 1.0f; }
__device__ inline size_t lora_at(int row, int n_ids, size_t id, size_t tok) {
    const int t = row / n_ids;
    return (size_t)t * tok + (size_t)(row - t * n_ids) * id;
}
__device__ inline const float* lora_x(const LoraArgs& a, int row) {
    const int t = row / a.n_ids, i = row - t * a.n_ids;
    return reinterpret_cast<const float*>(a.x + (size_t)t * a.x_tok + (size_t)(i % a.x_rows) * a.x_id);
}

// s[r] = A[r] . x for r below rk, one wave per r at a time
template <typename W>
__device__ inline void lora_shrink(const typename W::T* A, const float* x, int k, int rk, float* s) {
    const int v = (int)threadIdx.x & 63, wave = (int)threadIdx.x >> 6, nw = (int)blockDim.x >> 6;
    for (int r = wave; r < rk; r += nw) {
        float acc = 0.0f;
        for (int i = v; i < k; i += 64) acc = __builtin_fmaf(W::value(A[(size_t)r * k + i]), x[i], acc);
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) acc += __shfl_xor(acc, o);
        if (v == 0) s[r] = acc;
    }
    __syncthreads();
}

// ---------------------------------------------------------------------------
// Tiles: up to 16 rows of one key.  A workgroup with a thread for every row of the call finds its
// tile by itself (lora_tile); above, k_lora_group sorts each window of 1,024 rows by key
// and lists its tiles.
// ---------------------------------------------------------------------------
constexpr int kLoraTile = 16;
constexpr int kLoraWindow = 1024;

struct LoraTiles {
    const int* order;             // [windows * 1024]: rows by key, each window on its own; null: found by each workgroup
    const int4* items;            // [windows][slots]: (key, position in order, rows)
    const int* n_items;           // [windows]
    int n_rows, slots, skip_none; // skip_none: rows without an adapter are left alone
    int key_bits;                 // of key + 2 and of one more
    int cols;                     // columns of the output per workgroup
};

struct LoraGroup {
    int* order;
    int4* items;
    int* n_items;
    int n_rows, slots, skip_none, key_bits;
};

// A row's word, (key + 2, row of the window); past the rows one above every key
__device__ inline uint32_t lora_word(const LoraArgs& a, int row, int n_rows, int at) {
    if (row >= n_rows) return ((uint32_t)(a.n_adapters * a.n_experts + 2) << 10) | (uint32_t)at;
    const int key = lora_key(a, row);
    if (key == kLoraBad) *reinterpret_cast<volatile unsigned int*>(a.err) = kErrLora;
    return ((uint32_t)(key + 2) << 10) | (uint32_t)at;
}

// LDS of the sort: NW waves at most
template <int NW>
struct LoraSort {
    uint32_t c[64 * NW];
    int w[NW];                    // zeros for waves that the workgroup lacks
    uint64_t m[NW];
};

// The workgroup's words in the order of their keys (stable), one per thread, left in f.c too: a radix sort by single
// bits, as many as the keys have.  Every wave reads all the waves' counts at once: a loop over
// them cost 0.8 us a bit with 16 waves.
template <int NW>
__device__ inline uint32_t lora_sort(uint32_t c, int bits, LoraSort<NW>& f) {
    const int tid = (int)threadIdx.x, lane = tid & 63, wave = tid >> 6, nt = (int)blockDim.x;
    if (tid < NW) {
        f.w[tid] = 0;
        f.m[tid] = 0;
    }
    f.c[tid] = c;
    __syncthreads();
    for (int b = 10; b < 10 + bits; ++b) {
        const bool one = (c >> b) & 1u;
        const uint64_t m = __ballot(one);
        if (lane == 0) f.w[wave] = __popcll(m);
        __syncthreads();
        int ones = __popcll(m & ((1ull << lane) - 1ull)), total = 0;
#pragma unroll
        for (int v = 0; v < NW; ++v) {
            const int x = f.w[v];
            ones += v < wave ? x : 0;
            total += x;
        }
        f.c[one ? nt - total + ones : tid - ones] = c;
        __syncthreads();
        c = f.c[tid];
    }
    return c;
}

// In sorted order: every 16th row of a run of equal keys begins a tile.  The thread's tile, if it begins one
// (its number of rows, else 0), and the tiles before it.
template <int NW>
__device__ inline int lora_leader(uint32_t c, LoraSort<NW>& f, int n_keys2, bool skip_none, int& slot) {
    const int tid = (int)threadIdx.x, lane = tid & 63, wave = tid >> 6, nt = (int)blockDim.x;
    const uint32_t k2 = c >> 10;
    const uint64_t head = __ballot(tid == 0 || (f.c[max(tid - 1, 0)] >> 10) != k2);   // rows that begin a run
    if (lane == 0) f.m[wave] = head;
    __syncthreads();
    int start = 0;                                          // of the thread's run
    uint64_t next = 0;                                      // the heads of the wave after this one
#pragma unroll
    for (int v = 0; v < NW; ++v) {
        const uint64_t h = f.m[v];
        if (v < wave && h) start = 64 * v + 63 - __builtin_clzll(h);
        if (v == wave + 1) next = h;
    }
    const uint64_t upto = head & ((2ull << lane) - 1ull), after = head & ~((2ull << lane) - 1ull);
    if (upto) start = 64 * wave + 63 - __builtin_clzll(upto);
    int end = after ? 64 * wave + __builtin_ctzll(after) : next ? 64 * wave + 64 + __builtin_ctzll(next) : nt;
    const bool leader = (int)k2 < n_keys2 && ((tid - start) & (kLoraTile - 1)) == 0 && !(skip_none && (int)k2 == kLoraNone + 2);
    const uint64_t m = __ballot(leader);
    __syncthreads();
    if (lane == 0) f.w[wave] = __popcll(m);
    __syncthreads();
    slot = __popcll(m & ((1ull << lane) - 1ull));
#pragma unroll
    for (int v = 0; v < NW; ++v) slot += v < wave ? f.w[v] : 0;
    return leader ? min(kLoraTile, end - tid) : 0;          // a head two waves on is more than 16 rows away
}

// One window per workgroup, a row per thread.  Without atomics: the same rows give the same tiles.
__global__ __launch_bounds__(kLoraWindow) void k_lora_group(LoraArgs a, LoraGroup g) {
    __shared__ LoraSort<kLoraWindow / 64> f;
    const int tid = (int)threadIdx.x, w = (int)blockIdx.x, n_keys2 = a.n_adapters * a.n_experts + 2;
    const uint32_t c = lora_sort(lora_word(a, w * kLoraWindow + tid, g.n_rows, tid), g.key_bits, f);
    int slot;
    const int n = lora_leader(c, f, n_keys2, g.skip_none, slot);
    if (n) g.items[(size_t)w * g.slots + slot] = make_int4((int)(c >> 10) - 2, w * kLoraWindow + tid, n, 0);
    if (tid == (int)blockDim.x - 1) g.n_items[w] = slot + (n ? 1 : 0);
    if ((int)(c >> 10) < n_keys2) g.order[w * kLoraWindow + tid] = w * kLoraWindow + (int)(c & 1023u);
}

// LDS of a workgroup that finds its own tile
template <int NW>
struct LoraFind {
    LoraSort<NW> s;
    int item[3];
};

// The workgroup's tile: its key and number of rows, and the row of the lane's place
// lane % 16 in it (the last one's again past the number).  False: no tile is left for it.
template <int NW>
__device__ inline bool lora_tile(const LoraArgs& a, const LoraTiles& t, LoraFind<NW>& f, int& key, int& n, int& row) {
    const int tid = (int)threadIdx.x, p = tid & (kLoraTile - 1);
    if (t.order) {
        const int w = (int)blockIdx.z;
        if ((int)blockIdx.x >= t.n_items[w]) return false;
        const int4 it = t.items[(size_t)w * t.slots + blockIdx.x];
        key = __builtin_amdgcn_readfirstlane(it.x);
        n = __builtin_amdgcn_readfirstlane(it.z);
        row = t.order[it.y + min(p, n - 1)];
        return true;
    }
    if (t.n_rows == 1) {
        row = 0;
        n = 1;
        key = __builtin_amdgcn_readfirstlane(lora_key(a, 0));
        if (key == kLoraBad && tid == 0) *reinterpret_cast<volatile unsigned int*>(a.err) = kErrLora;
        return !(t.skip_none && key == kLoraNone);
    }
    const uint32_t c = lora_sort(lora_word(a, tid, t.n_rows, tid), t.key_bits, f.s);
    if (tid == 0) f.item[2] = 0;
    int slot;
    const int m = lora_leader(c, f.s, a.n_adapters * a.n_experts + 2, t.skip_none, slot);
    if (m && slot == (int)blockIdx.x) {
        f.item[0] = (int)(c >> 10) - 2;
        f.item[1] = tid;
        f.item[2] = m;
    }
    __syncthreads();
    n = __builtin_amdgcn_readfirstlane(f.item[2]);
    if (n == 0) return false;
    key = __builtin_amdgcn_readfirstlane(f.item[0]);
    row = (int)(f.s.c[f.item[1] + min(p, n - 1)] & 1023u);
    return true;
}

// columns c0 .. c1 of a tile whose rows have no adapter (a copy of base, or zeros) or a bad id (NaN)
__device__ inline void lora_plain_rows(const LoraArgs& a, int key, int n, int row, int c0, int c1) {
    for (int p = 0; p < n; ++p) {
        const int r = __shfl(row, p);
        float* dst = reinterpret_cast<float*>(a.dst + lora_at(r, a.n_ids, a.dst_id, a.dst_tok));
        const float* base =
            a.base ? reinterpret_cast<const float*>(a.base + lora_at(r, a.n_ids, a.base_id, a.base_tok)) : nullptr;
        for (int o = c0 + (int)threadIdx.x; o < c1; o += (int)blockDim.x)
            dst[o] = key == kLoraBad ? __builtin_nanf("") : base ? base[o] : 0.0f;
    }
}

// eight values of a row from column i on, zeros from column n on
template <typename W>
__device__ inline typename W::V8 lora_load8(const typename W::T* row, int i, int n) {
    if (i + 8 <= n) return W::load8(row + i);
    typename W::V8 v{};
#pragma unroll
    for (int c = 0; c < 8; ++c)
        if (i + c < n) W::set(v, c, row[i + c]);
    return v;
}

// ---------------------------------------------------------------------------
// Products of a weight operand (A: row m = lane % 16 of it) with an f32 operand (B: column lane % 16), eight
// neighbours of the summed axis per lane, on a tile whose lane holds column lane % 16 and rows 4 (lane / 16) .. +3.
//   f32 and f16 weights   eight v_mfma_f32_16x16x4 (any order of the summed axis is the same sum)
//   bf16 weights          the f32 operand in three bf16 pieces that add up to it exactly (each
//                         keeps the next 8 of its 24 bits), three v_mfma_f32_16x16x32_bf16: 48
//                         cycles against 256, with the same products and an f32 sum
// An infinity has no pieces (its rest is inf - inf): its columns are done with the f32 form (big).
// ---------------------------------------------------------------------------
typedef __bf16 lb8 __attribute__((ext_vector_type(8)));

struct LoraPieces {
    lb8 v[3];
};
__device__ inline LoraPieces lora_split(const float (&x)[8]) {
    union {
        uint32_t u[4];
        lb8 b;
    } p[3];
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        float r[2] = {x[2 * c], x[2 * c + 1]};
#pragma unroll
        for (int g = 0; g < 3; ++g) {
            // the upper halves of the two words
            p[g].u[c] = __builtin_amdgcn_perm(__float_as_uint(r[1]), __float_as_uint(r[0]), 0x07060302u);
#pragma unroll
            for (int e = 0; e < 2; ++e) r[e] = r[e] - __uint_as_float(__float_as_uint(r[e]) & 0xFFFF0000u);
        }
    }
    return LoraPieces{{p[0].b, p[1].b, p[2].b}};
}
__device__ inline float lora_most(const float (&x)[8], float m) {
#pragma unroll
    for (int c = 0; c < 8; ++c) m = fmaxf(m, __builtin_fabsf(x[c]));
    return m;
}
// lane p's flag of column p, from the four lanes that hold it
__device__ inline bool lora_column_big(float most) {
    most = fmaxf(most, __shfl_xor(most, 16));
    return fmaxf(most, __shfl_xor(most, 32)) == __builtin_inff();
}
template <typename W>
constexpr bool kLoraPieces = false;
template <>
constexpr bool kLoraPieces<LoraBF16> = true;

// S = X A^T of a tile: the waves share k in steps of 32, of which lane l holds the eight
// values at 8 (l / 16) of row l % 16 of X and of A; part [NW][16 NR][16] gets each wave's (rank, row).  Rows of
// A past the rank are the last one's again.  U steps are loaded while U others are multiplied.
template <typename W, int NR, int NW, int U>
struct LoraShrink {
    struct In {
        LoraF32::V8 x;
        typename W::V8 a[NR];
    };
    const typename W::T* ar[NR];
    const float* x;
    int k, q;
    float most = 0.0f;

    __device__ inline LoraShrink(const typename W::T* A, const float* x_, int k_, int rank) : x(x_), k(k_) {
        const int lane = (int)threadIdx.x & 63, p = lane & 15;
        q = lane >> 4;
#pragma unroll
        for (int b = 0; b < NR; ++b) ar[b] = A + (size_t)min(16 * b + p, rank - 1) * k;
    }
    __device__ inline void load(In& in, int s) const {
        const int i = s * 32 + 8 * q;
        in.x = LoraF32::load8(x + i);
#pragma unroll
        for (int b = 0; b < NR; ++b) in.a[b] = W::load8(ar[b] + i);
    }
    __device__ inline void load_rest(In& in, int s) const {
        const int i = s * 32 + 8 * q;
        in.x = lora_load8<LoraF32>(x, i, k);
#pragma unroll
        for (int b = 0; b < NR; ++b) in.a[b] = lora_load8<W>(ar[b], i, k);
    }
    template <bool PIECES>
    __device__ inline void mul(const In& in, lf4 (&acc)[NR]) {
        if constexpr (PIECES) {
            float v[8];
#pragma unroll
            for (int c = 0; c < 8; ++c) v[c] = LoraF32::get(in.x, c);
            most = lora_most(v, most);
            const LoraPieces P = lora_split(v);
#pragma unroll
            for (int g = 2; g >= 0; --g)
#pragma unroll
                for (int b = 0; b < NR; ++b)
                    acc[b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(lb8, in.a[b]), P.v[g], acc[b], 0, 0, 0);
        } else {
#pragma unroll
            for (int c = 0; c < 8; ++c)
#pragma unroll
                for (int b = 0; b < NR; ++b)
                    acc[b] = __builtin_amdgcn_mfma_f32_16x16x4f32(W::get(in.a[b], c), LoraF32::get(in.x, c), acc[b], 0, 0, 0);
        }
    }
    template <bool PIECES>
    __device__ inline void sum(lf4 (&acc)[NR]) {
        const int wave = (int)threadIdx.x >> 6, steps = k / 32;
#pragma unroll
        for (int b = 0; b < NR; ++b) acc[b] = lf4{0, 0, 0, 0};
        In in[2][U];
        auto load_all = [&](In (&z)[U], int s) {
#pragma unroll
            for (int u = 0; u < U; ++u) load(z[u], s + u * NW);
        };
        auto mul_all = [&](const In (&z)[U]) {
#pragma unroll
            for (int u = 0; u < U; ++u) mul<PIECES>(z[u], acc);
        };
        int s = wave;                                       // the first step that is not loaded
        auto more = [&] { return s + (U - 1) * NW < steps; };
        if (more()) {
            load_all(in[0], s);
            s += U * NW;
            for (;;) {
                bool m = more();
                if (m) load_all(in[1], s), s += U * NW;
                mul_all(in[0]);
                if (!m) break;
                m = more();
                if (m) load_all(in[0], s), s += U * NW;
                mul_all(in[1]);
                if (!m) break;
            }
        }
        for (; s <= steps; s += NW) {                       // what is left of whole steps, then k's rest
            if (s == steps && k % 32 == 0) break;
            load_rest(in[0][0], s);
            mul<PIECES>(in[0][0], acc);
        }
    }
    __device__ inline void run(float* part) {
        const int lane = (int)threadIdx.x & 63, wave = (int)threadIdx.x >> 6, p = lane & 15;
        lf4 acc[NR];
        sum<kLoraPieces<W>>(acc);
        if constexpr (kLoraPieces<W>) {
            if (__any(most == __builtin_inff())) {          // rare: the columns with an infinity again
                const bool big = lora_column_big(most);
                lf4 again[NR];
                sum<false>(again);
#pragma unroll
                for (int b = 0; b < NR; ++b)
#pragma unroll
                    for (int i = 0; i < 4; ++i) acc[b][i] = big ? again[b][i] : acc[b][i];
            }
        }
#pragma unroll
        for (int b = 0; b < NR; ++b)
#pragma unroll
            for (int i = 0; i < 4; ++i) part[((size_t)wave * 16 * NR + 16 * b + 4 * q + i) * 16 + p] = acc[b][i];
    }
};

// y = base + B S over columns c0 .. c1 of the tile, in steps of 32 columns per wave: D = B S^T, two products of 16
// columns, so that a lane holds eight neighbouring columns (four of each) of row lane % 16.
// The ranks of a lane's 4 NR values of a row of B and of S: groups of GW from 4 NR (lane / 16) on; a
// group that reaches past the rank is moved back to the row's last GW (rows of fewer than four: the
// last value again), so that loads stay inside the row.  A value counts if it is not one that an
// earlier group has, and below the adapter's own rank; the others' weights become zeros by a
// mask in registers (a NaN or an infinity past an adapter's own rank must not meet its zero in S).
template <typename W, int NR, int NW>
struct LoraExpand {
    static constexpr int GW = NR == 1 ? 4 : 8, NG = 4 * NR / GW;
    typedef typename std::conditional<NR == 1, typename W::V4, typename W::V8>::type V;
    struct In {
        V w[2][NG];
        lf4 y[2];
    };
    const typename W::T* B;
    const float* base;
    float* dst;
    int rank, rows, c1, p, q, at[NG];
    bool live;

    __device__ inline LoraExpand(const typename W::T* B_, int rank_, int rows_, const float* base_, float* dst_, bool live_,
                                 int c1_)
        : B(B_), base(base_), dst(dst_), rank(rank_), rows(rows_), c1(c1_), live(live_) {
        const int lane = (int)threadIdx.x & 63;
        p = lane & 15;
        q = lane >> 4;
#pragma unroll
        for (int g = 0; g < NG; ++g) at[g] = min(4 * NR * q + GW * g, max(0, rank - GW));
    }
    __device__ inline bool counts(int j, int rk) const {
        const int r = at[j / GW] + j % GW;
        return r >= 4 * NR * q + j / GW * GW && r < rk;
    }
    __device__ inline void load(In& in, int o0) const {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const typename W::T* row = B + (size_t)min(o0 + 8 * (p >> 2) + 4 * h + (p & 3), rows - 1) * rank;
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                if constexpr (NR == 1) {
                    if (rank < 4) {
#pragma unroll
                        for (int c = 0; c < 4; ++c) W::set(in.w[h][g], c, row[min(c, rank - 1)]);
                    } else {
                        in.w[h][g] = W::load4(row + at[g]);
                    }
                } else {
                    in.w[h][g] = W::load8(row + at[g]);
                }
            }
        }
        const int o = o0 + 8 * q;
        in.y[0] = lf4{0, 0, 0, 0};
        in.y[1] = lf4{0, 0, 0, 0};
        if (!base) return;
        if (o + 8 <= c1) {
            in.y[0] = *reinterpret_cast<const lf4u*>(base + o);
            in.y[1] = *reinterpret_cast<const lf4u*>(base + o + 4);
        } else {
#pragma unroll
            for (int c = 0; c < 8; ++c)
                if (o + c < c1) in.y[c >> 2][c & 3] = base[o + c];
        }
    }
    __device__ inline void store(const lf4 (&y)[2], int o0) const {
        const int o = o0 + 8 * q;
        if (!live) return;
        if (o + 8 <= c1) {
            *reinterpret_cast<lf4u*>(dst + o) = y[0];
            *reinterpret_cast<lf4u*>(dst + o + 4) = y[1];
        } else {
#pragma unroll
            for (int c = 0; c < 8; ++c)
                if (o + c < c1) dst[o + c] = y[c >> 2][c & 3];
        }
    }
    // in: the first step's, loaded by the caller (ahead of the shrink); s: the lane's S, already scaled, zeros
    // where a value does not count
    template <bool WHOLE>
    __device__ inline void run(In& in, int o0, const float (&s)[4 * NR], int rk) const {
        uint32_t mask[4 * NR];                              // of single values (f32 products), or pairs
        if constexpr (!WHOLE) {
#pragma unroll
            for (int j = 0; j < 4 * NR; ++j) {
                if constexpr (kLoraPieces<W>)
                    mask[j] = j % 2 ? 0 : (counts(j, rk) ? 0xFFFFu : 0u) | (counts(j + 1, rk) ? 0xFFFF0000u : 0u);
                else
                    mask[j] = counts(j, rk) ? 0xFFFFFFFFu : 0u;
                asm volatile("" : "+v"(mask[j]));           // kept as a word, not as a condition
            }
        }
        constexpr int NP = (NR + 1) / 2;                    // bf16 products of 32 ranks
        LoraPieces P[kLoraPieces<W> ? NP : 1];
        bool big = false, any_big = false;
        if constexpr (kLoraPieces<W>) {
            float most = 0.0f;
#pragma unroll
            for (int b = 0; b < NP; ++b) {
                float v[8];
#pragma unroll
                for (int c = 0; c < 8; ++c) v[c] = 8 * b + c < 4 * NR ? s[(8 * b + c) % (4 * NR)] : 0.0f;
                most = lora_most(v, most);
                P[b] = lora_split(v);
            }
            any_big = __any(most == __builtin_inff());
            if (any_big) big = lora_column_big(most);
        }
        auto weight = [&](const V& v, int g, int c) {
            const float w = W::get(v, c);
            if constexpr (WHOLE) return w;
            else if constexpr (kLoraPieces<W>)
                return __uint_as_float(__float_as_uint(w) & (mask[(GW * g + c) & ~1] << (c & 1 ? 0 : 16)) & 0xFFFF0000u);
            else return __uint_as_float(__float_as_uint(w) & mask[GW * g + c]);
        };
        auto f32_products = [&](const In& z, lf4 (&d)[2]) {
#pragma unroll
            for (int j = 0; j < 4 * NR; ++j)
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    d[h] = __builtin_amdgcn_mfma_f32_16x16x4f32(weight(z.w[h][j / GW], j / GW, j % GW), s[j], d[h], 0, 0, 0);
        };
        for (;;) {
            const int next = o0 + 32 * NW;
            In ahead;
            if (next < c1) load(ahead, next);
            lf4 d[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
            if constexpr (kLoraPieces<W>) {
#pragma unroll
                for (int b = 0; b < NP; ++b)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        union {
                            uint32_t u[4];
                            lb8 v;
                        } w;
                        if constexpr (NR == 1) {
                            const uint2 r = __builtin_bit_cast(uint2, in.w[h][0]);
                            w.u[0] = r.x, w.u[1] = r.y, w.u[2] = 0, w.u[3] = 0;
                        } else {
                            w.v = __builtin_bit_cast(lb8, in.w[h][b]);
                        }
                        if constexpr (!WHOLE) {
#pragma unroll
                            for (int c = 0; c < 4; ++c)
                                if (8 * b + 2 * c < 4 * NR) w.u[c] &= mask[(8 * b + 2 * c) % (4 * NR)];
                        }
#pragma unroll
                        for (int g = 2; g >= 0; --g) d[h] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w.v, P[b].v[g], d[h], 0, 0, 0);
                    }
                if (any_big) {
                    lf4 again[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
                    f32_products(in, again);
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int i = 0; i < 4; ++i) d[h][i] = big ? again[h][i] : d[h][i];
                }
            } else {
                f32_products(in, d);
            }
            const lf4 y[2] = {in.y[0] + d[0], in.y[1] + d[1]};
            store(y, o0);
            if (next >= c1) return;
            in = ahead;
            o0 = next;
        }
    }
};

// the lane's operand of S^T, of row lane % 16, times c; 0 where a value does not count
template <typename W, int NR, int NW>
__device__ inline void lora_sum_parts(const LoraExpand<W, NR, NW>& E, const float* part, int rk, float c, float (&s)[4 * NR]) {
    constexpr int GW = LoraExpand<W, NR, NW>::GW;
#pragma unroll
    for (int j = 0; j < 4 * NR; ++j) {
        const int r = E.at[j / GW] + j % GW;
        float v = 0.0f;
#pragma unroll
        for (int w = 0; w < NW; ++w) v += part[((size_t)w * 16 * NR + r) * 16 + E.p];
        s[j] = E.counts(j, rk) ? v * c : 0.0f;
    }
}

// One tile and t.cols columns per workgroup.  grid (slots, column parts, windows).
template <typename W, int NR, int NW, int U>
__global__ __launch_bounds__(64 * NW) void k_lora_apply(LoraArgs a, LoraTiles t) {
    __shared__ float part[NW * 16 * NR * 16];
    __shared__ LoraFind<NW> find;
    const int lane = (int)threadIdx.x & 63, wave = (int)threadIdx.x >> 6;
    int key, n, row;
    if (!lora_tile<NW>(a, t, find, key, n, row)) return;
    const int c0 = (int)blockIdx.y * t.cols, c1 = min(a.rows, c0 + t.cols), o0 = c0 + 32 * wave;
    if (key < 0) {
        lora_plain_rows(a, key, n, row, c0, c1);
        return;
    }
    const int rk = lora_rank(a, key);
    const float c = lora_scale(a, key);
    typedef LoraExpand<W, NR, NW> Expand;
    const Expand E(static_cast<const typename W::T*>(a.b) + (size_t)key * a.rows * a.rank, a.rank, a.rows,
                   a.base ? reinterpret_cast<const float*>(a.base + lora_at(row, a.n_ids, a.base_id, a.base_tok)) : nullptr,
                   reinterpret_cast<float*>(a.dst + lora_at(row, a.n_ids, a.dst_id, a.dst_tok)), (lane & 15) < n, c1);
    typename Expand::In in;
    if (o0 < c1) E.load(in, o0);
    LoraShrink<W, NR, NW, U>(static_cast<const typename W::T*>(a.a) + (size_t)key * a.rank * a.k, lora_x(a, row), a.k, a.rank)
        .run(part);
    __syncthreads();
    if (o0 >= c1) return;
    float s[4 * NR];
    lora_sum_parts(E, part, rk, c, s);
    if (rk == 16 * NR) E.template run<true>(in, o0, s, rk);
    else E.template run<false>(in, o0, s, rk);
}

// one workgroup per row: s, u and dx
template <typename W>
__global__ __launch_bounds__(kLoraThreads) void k_lora_back_rows(LoraArgs a) {
    __shared__ float s[kLoraMaxRank];
    __shared__ float u[kLoraMaxRank];
    const int row = (int)blockIdx.x, key = lora_key(a, row), tid = (int)threadIdx.x;
    float* dx = a.dx ? reinterpret_cast<float*>(a.dx + lora_at(row, a.n_ids, a.dx_id, a.dx_tok)) : nullptr;
    if (key < 0) {
        if (key == kLoraBad && tid == 0) *reinterpret_cast<volatile unsigned int*>(a.err) = kErrLora;
        if (dx && (key == kLoraBad || !a.add_dx))
            for (int i = tid; i < a.k; i += kLoraThreads) dx[i] = key == kLoraBad ? __builtin_nanf("") : 0.0f;
        return;
    }
    const int rk = lora_rank(a, key), v = tid & 63, wave = tid >> 6;
    const float c = lora_scale(a, key);
    const float* dy = reinterpret_cast<const float*>(a.dy + lora_at(row, a.n_ids, a.dy_id, a.dy_tok));
    const typename W::T* A = static_cast<const typename W::T*>(a.a) + (size_t)key * a.rank * a.k;
    const typename W::T* B = static_cast<const typename W::T*>(a.b) + (size_t)key * a.rows * a.rank;
    lora_shrink<W>(A, lora_x(a, row), a.k, rk, s);
    for (int r = wave; r < rk; r += kLoraThreads / 64) {
        float acc = 0.0f;
        for (int o = v; o < a.rows; o += 64) acc = __builtin_fmaf(W::value(B[(size_t)o * a.rank + r]), dy[o], acc);
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) acc += __shfl_xor(acc, o);
        if (v == 0) u[r] = c * acc;
    }
    __syncthreads();
    for (int r = tid; r < a.rank; r += kLoraThreads) {
        a.su[(size_t)row * 2 * a.rank + r] = r < rk ? s[r] : 0.0f;
        a.su[((size_t)row * 2 + 1) * a.rank + r] = r < rk ? u[r] : 0.0f;
    }
    if (!dx) return;
    for (int i = tid; i < a.k; i += kLoraThreads) {
        float acc = 0.0f;
        for (int r = 0; r < rk; ++r) acc = __builtin_fmaf(W::value(A[(size_t)r * a.k + i]), u[r], acc);
        dx[i] = a.add_dx ? dx[i] + acc : acc;
    }
}

// one workgroup per (key, r): dA[key][r] and dB[key][..][r], over the call's rows in order
__global__ __launch_bounds__(kLoraThreads) void k_lora_back_weights(LoraArgs a) {
    const int key = (int)blockIdx.x, r = (int)blockIdx.y, R = a.n_tokens * a.n_ids, tid = (int)threadIdx.x;
    const float c = lora_scale(a, key);
    float* da = a.da ? a.da + ((size_t)key * a.rank + r) * a.k : nullptr;
    float* db = a.db ? a.db + (size_t)key * a.rows * a.rank + r : nullptr;
    for (int i0 = 0; da && i0 < a.k; i0 += kLoraThreads) {
        const int i = i0 + tid;
        float acc = 0.0f;
        for (int row = 0; row < R; ++row)
            if (lora_key(a, row) == key && i < a.k)
                acc = __builtin_fmaf(a.su[((size_t)row * 2 + 1) * a.rank + r], lora_x(a, row)[i], acc);
        if (i < a.k) da[i] = a.add_dw ? da[i] + acc : acc;
    }
    for (int o0 = 0; db && o0 < a.rows; o0 += kLoraThreads) {
        const int o = o0 + tid;
        float acc = 0.0f;
        for (int row = 0; row < R; ++row)
            if (lora_key(a, row) == key && o < a.rows)
                acc = __builtin_fmaf(
                    a.su[(size_t)row * 2 * a.rank + r],
                    reinterpret_cast<const float*>(a.dy + lora_at(row, a.n_ids, a.dy_id, a.dy_tok))[o], acc);
        if (o < a.rows) db[(size_t)o * a.rank] = a.add_dw ? db[(size_t)o * a.rank] + c * acc : c * acc;
    }
}

}  // namespace sabah
