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
// Tiles: up to 16 rows of one key.  Up to 64 rows each workgroup finds its tile among
// them by itself (lora_tile); above, k_lora_group sorts each window of 1,024 rows by
// key and lists its tiles.
// ---------------------------------------------------------------------------
constexpr int kLoraTile = 16;
constexpr int kLoraDirectRows = 64;
constexpr int kLoraWindow = 1024;

struct LoraTiles {
    const int* order;             // [windows * 1024]: rows by key, each window on its own
    const int4* items;            // [windows][slots]: (key, position in order, rows)
    const int* n_items;           // [windows]
    int n_rows, slots, skip_none; // skip_none: rows without an adapter are left alone
    int cols;                     // columns of the output per workgroup
};

struct LoraGroup {
    int* order;
    int4* items;
    int* n_items;
    int n_rows, slots, skip_none;
};

// One window per workgroup: a bitonic sort of (key, row), a row per thread, in
// registers with the exchanges within a wave by shuffles; then every 16th row of a
// run of equal keys begins a tile.  Stable, and without atomics: the same rows
// give the same tiles.
__global__ __launch_bounds__(kLoraWindow) void k_lora_group(LoraArgs a, LoraGroup g) {
    __shared__ uint32_t s_c[kLoraWindow];
    __shared__ int s_w[kLoraWindow / 64];
    constexpr uint32_t kPad = 0xFFFFFFFFu;
    const int tid = (int)threadIdx.x, lane = tid & 63, wave = tid >> 6, w = (int)blockIdx.x;
    const int row = w * kLoraWindow + tid;
    uint32_t c = kPad;                                      // (key + 2, row of the window)
    if (row < g.n_rows) {
        const int key = lora_key(a, row);
        if (key == kLoraBad) *reinterpret_cast<volatile unsigned int*>(a.err) = kErrLora;
        c = ((uint32_t)(key + 2) << 10) | (uint32_t)tid;
    }
    for (int size = 2; size <= kLoraWindow; size <<= 1)
        for (int d = size >> 1; d > 0; d >>= 1) {
            uint32_t o;
            if (d < 64) {
                o = (uint32_t)__shfl_xor((int)c, d);
            } else {
                __syncthreads();
                s_c[tid] = c;
                __syncthreads();
                o = s_c[tid ^ d];
            }
            const bool lower = (tid & d) == 0, up = (tid & size) == 0;
            c = lower == up ? min(c, o) : max(c, o);
        }
    __syncthreads();
    s_c[tid] = c;
    __syncthreads();
    const bool valid = c != kPad;
    const uint32_t k2 = c >> 10;
    int start = tid > 0 && (s_c[tid - 1] >> 10) == k2 ? 0 : tid;   // the run's first thread: an inclusive maximum
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int y = __shfl_up(start, o);
        if (lane >= o) start = max(start, y);
    }
    if (lane == 63) s_w[wave] = start;
    __syncthreads();
    for (int v = 0; v < wave; ++v) start = max(start, s_w[v]);
    const bool leader = valid && ((tid - start) & (kLoraTile - 1)) == 0 && !(g.skip_none && (int)k2 - 2 == kLoraNone);
    const uint64_t m = __ballot(leader);
    __syncthreads();
    if (lane == 0) s_w[wave] = __popcll(m);
    __syncthreads();
    int slot = __popcll(m & ((1ull << lane) - 1ull));
    for (int v = 0; v < wave; ++v) slot += s_w[v];
    if (leader) {
        int n = 1;
        while (n < kLoraTile && tid + n < kLoraWindow && (s_c[tid + n] >> 10) == k2) ++n;
        g.items[(size_t)w * g.slots + slot] = make_int4((int)k2 - 2, w * kLoraWindow + tid, n, 0);
    }
    if (tid == kLoraWindow - 1) g.n_items[w] = slot + (leader ? 1 : 0);
    if (valid) g.order[w * kLoraWindow + tid] = w * kLoraWindow + (int)(c & 1023u);
}

// The workgroup's tile: its key and number of rows, and the row of the lane's place
// lane % 16 in it (the last one's again past the number).  False: no tile is left for it.
__device__ inline bool lora_tile(const LoraArgs& a, const LoraTiles& t, int lane, int& key, int& n, int& row) {
    const int p = lane & (kLoraTile - 1);
    if (t.order) {
        const int w = (int)blockIdx.z;
        if ((int)blockIdx.x >= t.n_items[w]) return false;
        const int4 it = t.items[(size_t)w * t.slots + blockIdx.x];
        key = __builtin_amdgcn_readfirstlane(it.x);
        n = __builtin_amdgcn_readfirstlane(it.z);
        row = t.order[it.y + min(p, n - 1)];
        return true;
    }
    const int k = lane < t.n_rows ? lora_key(a, lane) : 0x7FFFFFFF;
    if (k == kLoraBad) *reinterpret_cast<volatile unsigned int*>(a.err) = kErrLora;
    int idx = 0;                                            // earlier rows of the lane's key
    for (int j = 0; j < t.n_rows; ++j) idx += __builtin_amdgcn_readlane(k, j) == k && j < lane;
    const bool leader = lane < t.n_rows && (idx & (kLoraTile - 1)) == 0 && !(t.skip_none && k == kLoraNone);
    const uint64_t m = __ballot(leader);
    const uint64_t mine = __ballot(leader && __popcll(m & ((1ull << lane) - 1ull)) == (int)blockIdx.x);
    if (mine == 0) return false;
    const int first = __builtin_ctzll(mine);
    key = __builtin_amdgcn_readlane(k, first);
    const int i0 = __builtin_amdgcn_readlane(idx, first);
    const bool in = lane < t.n_rows && k == key && idx >= i0 && idx < i0 + kLoraTile;
    n = __popcll(__ballot(in));
    // the lane's number to its place in the tile; the others' to place 63, which nobody reads
    const int at = __builtin_amdgcn_ds_permute((in ? idx - i0 : 63) * 4, lane);
    row = __shfl(at, min(p, n - 1));
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

// S = X A^T of a tile with v_mfma_f32_16x16x4: the waves share k in steps of 32, of which lane l holds the eight
// values at 8 (l / 16) of row l % 16 of X (B operand) and of A (A operand), any order of k being
// the same sum; part [NW][16 NR][16] gets each wave's (rank, row).  Rows of A past the rank are
// the last one's again.
template <typename W, int NR, int NW, int U>
__device__ inline void lora_shrink_tile(const typename W::T* A, const float* x, int k, int rank, float* part) {
    const int lane = (int)threadIdx.x & 63, wave = (int)threadIdx.x >> 6, p = lane & 15, q = lane >> 4;
    const typename W::T* ar[NR];
#pragma unroll
    for (int b = 0; b < NR; ++b) ar[b] = A + (size_t)min(16 * b + p, rank - 1) * k;
    lf4 acc[NR];
#pragma unroll
    for (int b = 0; b < NR; ++b) acc[b] = lf4{0, 0, 0, 0};
    const int steps = k / 32;
    auto step = [&](const LoraF32::V8& xv, const typename W::V8 (&av)[NR]) {
#pragma unroll
        for (int c = 0; c < 8; ++c)
#pragma unroll
            for (int b = 0; b < NR; ++b)
                acc[b] = __builtin_amdgcn_mfma_f32_16x16x4f32(W::get(av[b], c), LoraF32::get(xv, c), acc[b], 0, 0, 0);
    };
    int s = wave;
    for (; s + (U - 1) * NW < steps; s += NW * U) {
        LoraF32::V8 xv[U];
        typename W::V8 av[U][NR];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = (s + u * NW) * 32 + 8 * q;
            xv[u] = LoraF32::load8(x + i);
#pragma unroll
            for (int b = 0; b < NR; ++b) av[u][b] = W::load8(ar[b] + i);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) step(xv[u], av[u]);
    }
    for (; s <= steps; s += NW) {                           // what is left of the unrolled steps, then k's rest
        const int i = s * 32 + 8 * q;
        if (s == steps && k % 32 == 0) break;
        typename W::V8 av[NR];
#pragma unroll
        for (int b = 0; b < NR; ++b) av[b] = lora_load8<W>(ar[b], i, k);
        step(lora_load8<LoraF32>(x, i, k), av);
    }
#pragma unroll
    for (int b = 0; b < NR; ++b)
#pragma unroll
        for (int i = 0; i < 4; ++i) part[((size_t)wave * 16 * NR + 16 * b + 4 * q + i) * 16 + p] = acc[b][i];
}

// The ranks of a lane's 4 NR values of a row of B and of S: groups of four from 4 NR (lane / 16) on; a
// group that reaches past the rank is moved back to the row's last four (rows of fewer than four: the
// last value again), so that loads stay inside the row.  A value counts if it is not one that an
// earlier group has, and below the adapter's own rank.
__device__ inline int lora_group_at(int r, int rank) { return min(r, max(0, rank - 4)); }
__device__ inline bool lora_counts(int r, int c, int rank, int rk) {
    const int at = lora_group_at(r, rank) + c;
    return at >= r && at < rk;
}

// the lane's operand of S^T, of row lane % 16, times c; 0 where a value does not count
template <int NR, int NW>
__device__ inline void lora_sum_parts(const float* part, int rank, int rk, float c, float (&s)[4 * NR]) {
    const int lane = (int)threadIdx.x & 63, p = lane & 15, q = lane >> 4;
#pragma unroll
    for (int j = 0; j < 4 * NR; ++j) {
        const int r0 = 4 * NR * q + (j & ~3), r = lora_group_at(r0, rank) + (j & 3);
        float v = 0.0f;
#pragma unroll
        for (int w = 0; w < NW; ++w) v += part[((size_t)w * 16 * NR + r) * 16 + p];
        s[j] = lora_counts(r0, j & 3, rank, rk) ? v * c : 0.0f;
    }
}

// The lane's 4 NR weights of a row of B.  WHOLE: every value counts; else the others become zeros by a
// mask in registers (a NaN or an infinity past an adapter's own rank must not meet its zero in S).
template <typename W, int NR, bool WHOLE>
struct LoraRow {
    int at[NR];
    uint32_t mask[WHOLE ? 1 : NR][4];
    bool small;
    __device__ inline LoraRow(int rank, int rk) {
        const int q = ((int)threadIdx.x & 63) >> 4;
        small = rank < 4;
#pragma unroll
        for (int g = 0; g < NR; ++g) {
            const int r = 4 * (NR * q + g);
            at[g] = lora_group_at(r, rank);
            if constexpr (!WHOLE) {
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    mask[g][c] = lora_counts(r, c, rank, rk) ? 0xFFFFFFFFu : 0u;
                    asm volatile("" : "+v"(mask[g][c]));    // kept as a word, not as a condition
                }
            }
        }
    }
    __device__ inline void load(const typename W::T* row, int rank, typename W::V4 (&v)[NR]) const {
#pragma unroll
        for (int g = 0; g < NR; ++g) {
            if (!WHOLE && NR == 1 && small) {
#pragma unroll
                for (int c = 0; c < 4; ++c) W::set(v[g], c, row[min(c, rank - 1)]);
            } else {
                v[g] = W::load4(row + at[g]);
            }
        }
    }
    __device__ inline float get(const typename W::V4 (&v)[NR], int j) const {
        const float w = W::get(v[j >> 2], j & 3);
        if constexpr (WHOLE) return w;
        else return __uint_as_float(__float_as_uint(w) & mask[j >> 2][j & 3]);
    }
};

// y = base + B S over columns c0 .. c1 of the tile: D = B S^T, so that a lane holds eight neighbouring
// columns (two products' four each) of row lane % 16
template <typename W, int NR, int NW, bool WHOLE>
__device__ inline void lora_expand_tile(const typename W::T* B, const float (&s)[4 * NR], int rank, int rk, int rows,
                                        const float* base, float* dst, bool live, int c0, int c1) {
    const int lane = (int)threadIdx.x & 63, wave = (int)threadIdx.x >> 6, p = lane & 15, q = lane >> 4;
    const LoraRow<W, NR, WHOLE> L(rank, rk);
    for (int o0 = c0 + 32 * wave; o0 < c1; o0 += 32 * NW) {
        typename W::V4 w[2][NR];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int o = min(o0 + 8 * (p >> 2) + 4 * h + (p & 3), rows - 1);
            L.load(B + (size_t)o * rank, rank, w[h]);
        }
        const int o = o0 + 8 * q;
        const bool full = o + 8 <= c1;
        lf4 y[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
        if (base) {
            if (full) {
                y[0] = *reinterpret_cast<const lf4u*>(base + o);
                y[1] = *reinterpret_cast<const lf4u*>(base + o + 4);
            } else {
#pragma unroll
                for (int c = 0; c < 8; ++c)
                    if (o + c < c1) y[c >> 2][c & 3] = base[o + c];
            }
        }
        lf4 d[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
#pragma unroll
        for (int j = 0; j < 4 * NR; ++j)
#pragma unroll
            for (int h = 0; h < 2; ++h)
                d[h] = __builtin_amdgcn_mfma_f32_16x16x4f32(L.get(w[h], j), s[j], d[h], 0, 0, 0);
#pragma unroll
        for (int h = 0; h < 2; ++h) y[h] = y[h] + d[h];
        if (!live) continue;
        if (full) {
            *reinterpret_cast<lf4u*>(dst + o) = y[0];
            *reinterpret_cast<lf4u*>(dst + o + 4) = y[1];
        } else {
#pragma unroll
            for (int c = 0; c < 8; ++c)
                if (o + c < c1) dst[o + c] = y[c >> 2][c & 3];
        }
    }
}

// One tile and t.cols columns per workgroup.  grid (slots, column parts, windows).
template <typename W, int NR, int NW, int U>
__global__ __launch_bounds__(64 * NW) void k_lora_apply(LoraArgs a, LoraTiles t) {
    __shared__ float part[NW * 16 * NR * 16];
    const int lane = (int)threadIdx.x & 63;
    int key, n, row;
    if (!lora_tile(a, t, lane, key, n, row)) return;
    const int c0 = (int)blockIdx.y * t.cols, c1 = min(a.rows, c0 + t.cols);
    if (key < 0) {
        lora_plain_rows(a, key, n, row, c0, c1);
        return;
    }
    const int rk = lora_rank(a, key);
    const float c = lora_scale(a, key);
    lora_shrink_tile<W, NR, NW, U>(static_cast<const typename W::T*>(a.a) + (size_t)key * a.rank * a.k, lora_x(a, row), a.k,
                                   a.rank, part);
    __syncthreads();
    float s[4 * NR];
    lora_sum_parts<NR, NW>(part, a.rank, rk, c, s);
    const typename W::T* B = static_cast<const typename W::T*>(a.b) + (size_t)key * a.rows * a.rank;
    const float* base =
        a.base ? reinterpret_cast<const float*>(a.base + lora_at(row, a.n_ids, a.base_id, a.base_tok)) : nullptr;
    float* dst = reinterpret_cast<float*>(a.dst + lora_at(row, a.n_ids, a.dst_id, a.dst_tok));
    const bool live = (lane & 15) < n;
    if (rk == 16 * NR) lora_expand_tile<W, NR, NW, true>(B, s, a.rank, rk, a.rows, base, dst, live, c0, c1);
    else lora_expand_tile<W, NR, NW, false>(B, s, a.rank, rk, a.rows, base, dst, live, c0, c1);
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
