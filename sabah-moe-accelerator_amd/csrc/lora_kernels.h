// Low-rank adapters of many requests beside a shared projection, and their
// gradients.  Row r is (token t, slot i); its adapter is adapters[t] (-1: none)
// and its expert ids[t][i] (0 without ids); A and B are the pair of that key.
//   forward    s = A x_r;  y_r = base_r + scale B s
//   backward   u = scale B^T dy_r;  dx_r (+)= A^T u;  dA (+)= u x_r^T;  dB (+)= scale dy_r s^T
// Sums are f32; weights of f16 and bf16 are widened exactly.
#pragma once
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

namespace sabah {

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
    const int e = a.ids ? *reinterpret_cast<const int32_t*>(a.ids + (size_t)t * a.ids_tok + (size_t)i * a.ids_id) : 0;
    if (ad == -1) return kLoraNone;
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

// ---------------------------------------------------------------------------
// Tiles: up to 16 rows of one key.  In small calls each workgroup finds its tile by itself
// (lora_tile, a thread for every row of the call); above, k_lora_group sorts each window of 1,024
// rows by key and lists its tiles.
// ---------------------------------------------------------------------------
// A tile of the lists is one sixteen of rows forward, two backward (LoraGroup::tile).  Two share the reads of A and B, which
// pays where the weights' gradients take whole tiles of 32 anyway; forward, half as many workgroups cost more: 1,999
// rows at rank 64 21.7 us in sixteens, 23.6 in twos; at rank 128 33 and 45; 16,384 rows at rank 64 96 and 93, at 128 154 and 162.
constexpr int kLoraTile = 16;
constexpr int kLoraWindow = 1024;

struct LoraTiles {
    const int* order;             // [windows * 1024]: rows by key, each window on its own
    const int4* items;            // [windows][slots]: (key, position in order, rows)
    const int* n_items;           // [windows]
    int n_rows, slots, skip_none; // skip_none: rows without an adapter are left alone
    int key_bits;                 // of key + 2 and of one more
    int cols;                     // columns of the output per workgroup
    float* s;                     // larger calls: [k_parts][positions][rank, in 16s]
    int k_parts, k_steps, positions;
    uint16_t* pieces;             // backward, one k part: [windows * slots][3 pieces][rank, in 16s][32 rows] of s, or null
    uint64_t* off;                // with pieces: [windows * slots][32], the rows' byte offsets in x
    int scaled;                   // pieces of c s
};

struct LoraGroup {
    int* order;
    int4* items;
    int* n_items;
    int n_rows, slots, skip_none, key_bits, tile;
    uint32_t* runs;               // or [windows][keys]: a key's rows in the window << 16 | its first tile's slot, 0 without any
};

// A row's word, (key + 2, row of the window); past the rows one above every key
__device__ inline uint32_t lora_word(const LoraArgs& a, int row, int n_rows, int at) {
    if (row >= n_rows) return ((uint32_t)(a.n_adapters * a.n_experts + 2) << 10) | (uint32_t)at;
    const int key = lora_key(a, row);
    if (key == kLoraBad) *reinterpret_cast<volatile unsigned int*>(a.err) = kErrLora;
    return ((uint32_t)(key + 2) << 10) | (uint32_t)at;
}

// LDS of the sort: NW waves at most (16); w and m are zeros for waves that the workgroup lacks
template <int NW>
struct LoraSort {
    uint32_t c[64 * NW];
    uint2 w[16];
    uint64_t m[NW + 1];
};

// inclusive sum over the 16 lanes of a row up to the lane's
__device__ inline uint32_t lora_row_scan(uint32_t v) {
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x111, 0xF, 0xF, true);     // row_shr 1, 2, 4, 8
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x112, 0xF, 0xF, true);
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x114, 0xF, 0xF, true);
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x118, 0xF, 0xF, true);
    return v;
}

// The workgroup's words in the order of their keys (stable), one per thread, left in f.c too: a radix sort by two
// bits, as many as the keys have.  A wave's counts of the four digits are packed in four halves, and
// every wave sums all the waves' in its lanes (a loop over them cost 0.8 us a bit with 16 waves).
template <int NW>
__device__ inline uint32_t lora_sort(uint32_t c, int bits, LoraSort<NW>& f) {
    const int tid = (int)threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    if (tid < 16) f.w[tid] = make_uint2(0, 0);
    if (tid <= NW) f.m[tid] = 0;
    f.c[tid] = c;
    __syncthreads();
    for (int b = 10; b < 10 + bits; b += 2) {
        const uint32_t d = (c >> b) & 3u;
        const uint64_t hi = __ballot((d & 2u) != 0), lo = __ballot((d & 1u) != 0);
        const uint2 own = make_uint2((uint32_t)__popcll(~hi & ~lo) | (uint32_t)__popcll(~hi & lo) << 16,
                                     (uint32_t)__popcll(hi & ~lo) | (uint32_t)__popcll(hi & lo) << 16);
        if (lane == 0) f.w[wave] = own;
        __syncthreads();
        const uint2 x = f.w[lane & 15];
        const uint32_t sx = lora_row_scan(x.x), sy = lora_row_scan(x.y);
        const uint32_t tx = (uint32_t)__builtin_amdgcn_readlane((int)sx, 15), ty = (uint32_t)__builtin_amdgcn_readlane((int)sy, 15);
        const uint32_t bx = (uint32_t)__builtin_amdgcn_readlane((int)sx, wave) - own.x,
                       by = (uint32_t)__builtin_amdgcn_readlane((int)sy, wave) - own.y;
        const uint32_t n0 = tx & 0xFFFFu, n1 = n0 + (tx >> 16), n2 = n1 + (ty & 0xFFFFu);
        const uint64_t same = (d & 2u ? hi : ~hi) & (d & 1u ? lo : ~lo);
        const uint32_t first = d & 2u ? (d & 1u ? n2 + (by >> 16) : n1 + (by & 0xFFFFu)) : d & 1u ? n0 + (bx >> 16) : bx & 0xFFFFu;
        f.c[first + (uint32_t)__popcll(same & ((1ull << lane) - 1ull))] = c;
        __syncthreads();
        c = f.c[tid];
    }
    return c;
}

// In sorted order: every 16th (or tile-th) row of a run of equal keys begins a tile.  The thread's tile, if it begins one
// (its number of rows, else 0), and the tiles before it.
template <int NW>
__device__ inline int lora_leader(uint32_t c, LoraSort<NW>& f, int n_keys2, bool skip_none, int& slot, int tile = kLoraTile, int* run = nullptr) {
    const int tid = (int)threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), nt = (int)blockDim.x;
    const uint32_t k2 = c >> 10;
    const uint64_t head = __ballot(tid == 0 || (f.c[max(tid - 1, 0)] >> 10) != k2);   // rows that begin a run
    __syncthreads();
    if (lane == 0) {
        f.m[wave] = head;
        f.w[wave].x = head ? 64u * wave + 63u - (uint32_t)__builtin_clzll(head) : 0u;
    }
    __syncthreads();
    // the last head of the earlier waves
    const uint64_t next = f.m[wave + 1];
    const uint32_t last = f.w[lane & 15].x;
    const uint64_t upto = head & ((2ull << lane) - 1ull), after = head & ~((2ull << lane) - 1ull);
    int start = 0;
#pragma unroll
    for (int v = 0; v < NW; ++v) start = max(start, v < wave ? __builtin_amdgcn_readlane((int)last, v) : 0);
    if (upto) start = 64 * wave + 63 - __builtin_clzll(upto);
    const int end = after ? 64 * wave + __builtin_ctzll(after) : next ? 64 * wave + 64 + __builtin_ctzll(next) : nt;
    const bool leader = (int)k2 < n_keys2 && ((tid - start) & (tile - 1)) == 0 && !(skip_none && (int)k2 == kLoraNone + 2);
    const uint64_t m = __ballot(leader);
    __syncthreads();
    if (lane == 0) f.w[wave].x = (uint32_t)__popcll(m);
    __syncthreads();
    const uint32_t before = lora_row_scan(f.w[lane & 15].x);
    slot = __builtin_amdgcn_readlane((int)before, wave) - __popcll(m) + __popcll(m & ((1ull << lane) - 1ull));
    if (run) {                                              // of the threads that begin one, the whole run's rows
        int stop = after || next ? end : nt;
        for (int v = wave + 2; v < NW && !after && !next; ++v)
            if (f.m[v]) {
                stop = 64 * v + __builtin_ctzll(f.m[v]);
                break;
            }
        *run = leader && tid == start ? stop - tid : 0;
    }
    return leader ? min(tile, end - tid) : 0;               // a head two waves on is more than a tile away
}

// One window per workgroup, a row per thread.  Without atomics: the same rows give the same tiles.
__global__ __launch_bounds__(kLoraWindow) void k_lora_group(LoraArgs a, LoraGroup g) {
    __shared__ LoraSort<kLoraWindow / 64> f;
    const int tid = (int)threadIdx.x, w = (int)blockIdx.x, n_keys2 = a.n_adapters * a.n_experts + 2;
    const uint32_t c = lora_sort(lora_word(a, w * kLoraWindow + tid, g.n_rows, tid), g.key_bits, f);
    if (g.runs)
        for (int i = tid; i < n_keys2 - 2; i += (int)blockDim.x) g.runs[(size_t)w * (n_keys2 - 2) + i] = 0u;
    int slot, run;
    const int n = lora_leader(c, f, n_keys2, g.skip_none, slot, g.tile, &run);     // its barriers order the zeros before the runs
    if (g.runs && run && (int)(c >> 10) >= 2)
        g.runs[(size_t)w * (n_keys2 - 2) + (c >> 10) - 2] = (uint32_t)run << 16 | (uint32_t)slot;
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
__device__ inline bool lora_tile(const LoraArgs& a, const LoraTiles& t, LoraFind<NW>& f, int& key, int& n, int (&rows)[1]) {
    int& row = rows[0];
    const int tid = (int)threadIdx.x, p = tid & (kLoraTile - 1);
    if (t.n_rows == 1) {
        row = 0;
        n = 1;
        key = __builtin_amdgcn_readfirstlane(lora_key(a, 0));
        if (key == kLoraBad && tid == 0) *reinterpret_cast<volatile unsigned int*>(a.err) = kErrLora;
        return !(t.skip_none && key == kLoraNone);
    }
    if (t.n_rows <= 64) {                                   // every wave for itself, without a barrier
        const int lane = tid & 63, k = lane < t.n_rows ? lora_key(a, lane) : 0x7FFFFFFF;
        if (k == kLoraBad) *reinterpret_cast<volatile unsigned int*>(a.err) = kErrLora;
        int idx = 0;                                        // earlier rows of the lane's key
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

// The same from the lists of k_lora_group, with the tile's position in order; row[h]: of place h0 + 16 h + lane % 16
template <int H>
__device__ inline bool lora_item(const LoraTiles& t, int w, int& key, int& n, int (&row)[H], int& pos, int h0 = 0) {
    if ((int)blockIdx.x >= t.n_items[w]) return false;
    const int4 it = t.items[(size_t)w * t.slots + blockIdx.x];
    key = __builtin_amdgcn_readfirstlane(it.x);
    pos = __builtin_amdgcn_readfirstlane(it.y);
    n = __builtin_amdgcn_readfirstlane(it.z);
#pragma unroll
    for (int h = 0; h < H; ++h) row[h] = t.order[pos + min(h0 + 16 * h + ((int)threadIdx.x & 15), n - 1)];
    return true;
}

// columns c0 .. c1 of a tile whose rows have no adapter (a copy of base, or zeros) or a bad id (NaN)
template <int H>
__device__ inline void lora_plain_rows(const LoraArgs& a, int key, int n, const int (&row)[H], int c0, int c1) {
    for (int p = 0; p < n; ++p) {
        const int r = __shfl(H == 1 || p < 16 ? row[0] : row[H - 1], p & 15);
        float* dst = reinterpret_cast<float*>(a.dst + lora_at(r, a.n_ids, a.dst_id, a.dst_tok));
        const float* base =
            a.base ? reinterpret_cast<const float*>(a.base + lora_at(r, a.n_ids, a.base_id, a.base_tok)) : nullptr;
        for (int o = c0 + (int)threadIdx.x; o < c1; o += (int)blockDim.x)
            dst[o] = key == kLoraBad ? __builtin_nanf("") : base ? base[o] : 0.0f;
    }
}

// ---------------------------------------------------------------------------
// Products of a weight operand with an f32 operand, eight neighbours of the summed axis per lane, on a 16 x 16 tile.
//   f32 weights    eight v_mfma_f32_16x16x4 (any order of the summed axis is the same sum): 256 cycles
//   bf16 weights   the f32 operand in three bf16 pieces that add up to it exactly (each keeps the next 8 of
//                  its 24 bits), three v_mfma_f32_16x16x32_bf16: 48 cycles, the same products
//   f16 weights    two f16 pieces of 11 bits, rounded to nearest, of the operand scaled by a power of two that
//                  brings its row's largest of these values to 2^14 .. 2^15: what is left out is at most
//                  2^-23 of a value.  32 cycles, and a product with the scale.  Below 2^-2 f16's exponents end: at
//                  2^-4, 2^-18 of the largest, up to 2^-21 is left out, and below that all may be (the instruction also
//                  aligns its products to the largest's, even where that one's weight is 0).  Rows with
//                  values below 2^-4 take the f32 form, about one step of 16 rows in four hundred of normally distributed
//                  values (with 2^-2 for the line, one in a hundred, 1,999 rows at rank 64 took 30.5 us, with 2^-4 28.9;
//                  28.3 without any).  Which they are goes by the row alone: its sums are the same whichever
//                  rows are beside it
// Sums are f32.  An infinity has no pieces (its rest is inf - inf), and one of the weights meets pieces that are 0: sums that
// come out as NaN are done again in the f32 form.
// ---------------------------------------------------------------------------
typedef __bf16 lb8 __attribute__((ext_vector_type(8)));
typedef _Float16 lh2 __attribute__((ext_vector_type(2)));
typedef _Float16 lh8 __attribute__((ext_vector_type(8)));
typedef float lf2 __attribute__((ext_vector_type(2)));

template <typename W>
constexpr int kLoraPieces = 0;                              // pieces of the f32 operand; 0: it stays whole
template <>
constexpr int kLoraPieces<LoraBF16> = 3;
template <>
constexpr int kLoraPieces<LoraF16> = 2;

struct LoraWords {
    uint32_t u[4];                                          // eight 16-bit values
};
__device__ inline lf4 lora_mfma(LoraBF16, const LoraWords& a, const LoraWords& b, lf4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(lb8, a), __builtin_bit_cast(lb8, b), c, 0, 0, 0);
}
__device__ inline lf4 lora_mfma(LoraF16, const LoraWords& a, const LoraWords& b, lf4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(lh8, a), __builtin_bit_cast(lh8, b), c, 0, 0, 0);
}
__device__ inline void lora_split(LoraBF16, const float (&x)[8], float, LoraWords (&w)[3]) {
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        float r[2] = {x[2 * c], x[2 * c + 1]};
#pragma unroll
        for (int g = 0; g < 3; ++g) {
            // the upper halves of the two words
            w[g].u[c] = __builtin_amdgcn_perm(__float_as_uint(r[1]), __float_as_uint(r[0]), 0x07060302u);
#pragma unroll
            for (int e = 0; e < 2; ++e) r[e] = r[e] - __uint_as_float(__float_as_uint(r[e]) & 0xFFFF0000u);
        }
    }
}
// Returns whether some value is small: not 0, and below 2^-4
__device__ inline bool lora_split(LoraF16, const float (&x)[8], float scale, LoraWords (&w)[2]) {
    uint32_t least = 0xFFFFFFFFu;                           // of the magnitudes' words times two less one: a 0 is the largest
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        lf2 r = {x[2 * c] * scale, x[2 * c + 1] * scale};
#pragma unroll
        for (int e = 0; e < 2; ++e) least = min(least, 2u * __float_as_uint(r[e]) - 1u);
#pragma unroll
        for (int g = 0; g < 2; ++g) {
            const lh2 h = __builtin_convertvector(r, lh2);
            w[g].u[c] = __builtin_bit_cast(uint32_t, h);
            r[0] = r[0] - (float)h[0];                      // exact
            r[1] = r[1] - (float)h[1];
        }
    }
    return least < 2u * 0x3D800000u - 1u;
}
// value c of eight 16-bit ones
template <typename W>
__device__ inline float lora_value(const LoraWords& w, int c) {
    return W::value((uint16_t)(c & 1 ? w.u[c / 2] >> 16 : w.u[c / 2] & 0xFFFFu));
}
// The power of two that brings `most` to 2^14 .. 2^15 (at most 2^126), and its inverse
__device__ inline float lora_scale_of(float most, float& back) {
    const uint32_t e = max(__float_as_uint(most) >> 23, 15u);
    back = __uint_as_float((e - 14u) << 23);
    return __uint_as_float((268u - e) << 23);
}
template <int N>
__device__ inline float lora_most(const float (&x)[N], float m) {
#pragma unroll
    for (int c = 0; c < N; ++c) m = fmaxf(m, __builtin_fabsf(x[c]));
    return m;
}
// of column p, from the four lanes that hold it
__device__ inline float lora_column_most(float most) {
    const uint32_t m = __float_as_uint(most);
    const auto h = __builtin_amdgcn_permlane32_swap(m, m, false, false);    // both halves in both
    const uint32_t n = max(h[0], h[1]);                                     // magnitudes order as words
    const auto r = __builtin_amdgcn_permlane16_swap(n, n, false, false);
    return __uint_as_float(max(r[0], r[1]));
}
// the rows (columns) that lanes of a ballot hold
__device__ inline unsigned lora_rows_of(uint64_t lanes) {
    lanes |= lanes >> 32;
    return (unsigned)(lanes | lanes >> 16) & 0xFFFFu;
}

// Two values' next bf16 piece, to nearest, packed, and their rests.  Three such pieces are within 2^-24 of a value, and so
// are the six products that k_lora_grad keeps of two values' nine.
__device__ inline uint32_t lora_split2(float (&v)[2]) {
    typedef __bf16 lb2 __attribute__((ext_vector_type(2)));
    const uint32_t h = __builtin_bit_cast(uint32_t, __builtin_convertvector((lf2{v[0], v[1]}), lb2));
    v[0] = v[0] - __uint_as_float(h << 16);
    v[1] = v[1] - __uint_as_float(h & 0xFFFF0000u);
    return h;
}

// S = X A^T of a tile: the waves share k in steps of 32, of which lane l's operands are the eight
// values at 8 (l / 16) of row l % 16 of X and of A.  Both are read along their rows and turned in LDS: in operand
// order neighbouring lanes read different rows, and the L1 takes 64 cycles a load instead of 16.
// part [NW][16 NR][17] gets each wave's (rank, row).  Rows of A past the rank are the last one's again.
// U steps are loaded at a time.
constexpr int kLoraPart = 17;                 // floats of part per rank
constexpr int kLoraXLds = 16 * 9;             // of a wave: 16 rows of 128 bytes, 144 apart: no bank conflicts either way
template <typename W>
constexpr int kLoraALds = sizeof(typename W::T) == 4 ? 16 * 9 : 16 * 4;   // rows of 128 bytes, or of 64 with their quarters exchanged
template <typename W, int NR, int NW, int U, int H>
struct LoraShrink {
    static constexpr int CH = sizeof(typename W::T) / 2;    // loads of 16 bytes for 16 rows of A
    struct In {
        lf4 x[H][2], a[NR][CH];
    };
    const typename W::T* A;
    const float* xr[H][2];
    uint32_t at[NR][CH];                                    // elements; rank * k is below 2^28
    lf4 *lx, *la;                                           // the wave's
    int k, s0, steps, p, q, lane, rank;                     // whole steps s0 .. steps, and k's rest if steps is the last
    bool second;                                            // the tile has more than 16 rows
    lf4 acc[H][NR];

    // row: of the lane's places lane % 16 in the tile of n rows; lds: NW * (kLoraXLds + kLoraALds<W>); of k the steps from s0
    // on, below s1
    __device__ inline LoraShrink(const LoraArgs& a, const typename W::T* A_, const int (&row)[H], int n, lf4* lds, int s0_, int s1)
        : A(A_), k(a.k), s0(s0_), steps(min(s1, a.k / 32)), rank(a.rank), second(H > 1 && n > 16) {
        lane = (int)threadIdx.x & 63;
        p = lane & 15;
        q = lane >> 4;
        lx = lds + ((int)threadIdx.x >> 6) * (kLoraXLds + kLoraALds<W>);
        la = lx + kLoraXLds;
#pragma unroll
        for (int t = 0; t < H; ++t)
#pragma unroll
            for (int h = 0; h < 2; ++h) xr[t][h] = lora_x(a, __shfl(row[t], 8 * h + (lane >> 3)));
#pragma unroll
        for (int b = 0; b < NR; ++b)
#pragma unroll
            for (int h = 0; h < CH; ++h) at[b][h] = (uint32_t)min(16 * b + a_row(h), a.rank - 1) * (uint32_t)k + a_col();
    }
    // of 16 rows of A in one step of 32 columns, the row and the first column of the lane's load h
    __device__ inline int a_row(int h) const { return CH == 1 ? lane >> 2 : 8 * h + (lane >> 3); }
    __device__ inline int a_col() const { return CH == 1 ? 8 * (lane & 3) : 4 * (lane & 7); }
    __device__ inline void load(In& in, int s) const {
#pragma unroll
        for (int t = 0; t < H; ++t)
            if (t == 0 || second) {
#pragma unroll
                for (int h = 0; h < 2; ++h) in.x[t][h] = *reinterpret_cast<const lf4u*>(xr[t][h] + s * 32 + 4 * (lane & 7));
            }
#pragma unroll
        for (int b = 0; b < NR; ++b)
#pragma unroll
            for (int h = 0; h < CH; ++h) {
                const typename W::T* w = A + at[b][h] + (uint32_t)s * 32u;
                if constexpr (CH == 1) in.a[b][h] = __builtin_bit_cast(lf4, W::load8(w));
                else in.a[b][h] = W::load4(w).v;
            }
    }
    __device__ inline void load_rest(In& in, int s) const {
        const int j = s * 32 + 4 * (lane & 7), i = s * 32 + a_col();
        constexpr int N = 16 / sizeof(typename W::T);
#pragma unroll
        for (int t = 0; t < H; ++t)
            if (t == 0 || second) {
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int c = 0; c < 4; ++c) in.x[t][h][c] = j + c < k ? xr[t][h][j + c] : 0.0f;
            }
#pragma unroll
        for (int b = 0; b < NR; ++b)
#pragma unroll
            for (int h = 0; h < CH; ++h) {
                union {
                    typename W::T t[N];
                    lf4 v;
                } w;
#pragma unroll
                for (int c = 0; c < N; ++c) w.t[c] = i + c < k ? A[at[b][h] + (uint32_t)(s * 32 + c)] : (typename W::T)0;
                in.a[b][h] = w.v;
            }
    }
    // 16 rows from the order of their loads to the operand's, eight values per lane.  The reads wait for the
    // writes (one wave, LDS in order); the barriers keep the compiler from moving either.
    __device__ inline void turn_rows128(lf4* lds, const lf4 (&in)[2], lf4 (&v)[2]) const {
#pragma unroll
        for (int h = 0; h < 2; ++h) lds[(8 * h + (lane >> 3)) * 9 + (lane & 7)] = in[h];
        __builtin_amdgcn_wave_barrier();
        v[0] = lds[p * 9 + 2 * q];
        v[1] = lds[p * 9 + 2 * q + 1];
        __builtin_amdgcn_wave_barrier();
    }
    __device__ inline lf4 turn_rows64(lf4* lds, const lf4& in) const {
        lds[(lane & ~3) + ((lane & 3) ^ ((lane >> 3) & 3))] = in;           // row lane / 4
        __builtin_amdgcn_wave_barrier();
        const lf4 v = lds[4 * p + (q ^ ((p >> 1) & 3))];
        __builtin_amdgcn_wave_barrier();
        return v;
    }
    __device__ inline void mul(const In& in) {
        if constexpr (kLoraPieces<W> > 0) {
            LoraWords w[NR];
#pragma unroll
            for (int b = 0; b < NR; ++b) w[b] = __builtin_bit_cast(LoraWords, turn_rows64(la, in.a[b][0]));
#pragma unroll
            for (int t = 0; t < H; ++t) {
                if (t > 0 && !second) continue;
                lf4 x[2];
                turn_rows128(lx, in.x[t], x);
                float v[8];
#pragma unroll
                for (int c = 0; c < 8; ++c) v[c] = x[c >> 2][c & 3];
                float back = 1.0f, scale = 1.0f;
                if constexpr (std::is_same<W, LoraF16>::value) scale = lora_scale_of(lora_column_most(lora_most(v, 0.0f)), back);
                LoraWords P[kLoraPieces<W>];
                if constexpr (std::is_same<W, LoraF16>::value) {
                    const bool some = lora_split(W{}, v, scale, P);
                    lf4 d[NR];
#pragma unroll
                    for (int b = 0; b < NR; ++b) d[b] = lf4{0, 0, 0, 0};
#pragma unroll
                    for (int g = kLoraPieces<W> - 1; g >= 0; --g)
#pragma unroll
                        for (int b = 0; b < NR; ++b) d[b] = lora_mfma(W{}, w[b], P[g], d[b]);
                    if (__builtin_expect(__any(some), 0)) {
                        __builtin_amdgcn_wave_barrier();
                        const bool mine = (lora_rows_of(__ballot(some)) >> p) & 1u;
                        if (mine) back = 1.0f;
                        const lf4 y[2] = {lx[p * 9 + 2 * q], lx[p * 9 + 2 * q + 1]};    // x again, not kept until here
#pragma unroll
                        for (int b = 0; b < NR; ++b) {
                            lf4 e = {0, 0, 0, 0};
#pragma unroll
                            for (int c = 0; c < 8; ++c)
                                e = __builtin_amdgcn_mfma_f32_16x16x4f32(lora_value<W>(w[b], c), y[c >> 2][c & 3], e, 0, 0, 0);
#pragma unroll
                            for (int i = 0; i < 4; ++i) d[b][i] = mine ? e[i] : d[b][i];
                        }
                        __builtin_amdgcn_wave_barrier();
                    }
#pragma unroll
                    for (int b = 0; b < NR; ++b)
#pragma unroll
                        for (int i = 0; i < 4; ++i) acc[t][b][i] = __builtin_fmaf(d[b][i], back, acc[t][b][i]);
                } else {
                    lora_split(W{}, v, scale, P);
#pragma unroll
                    for (int g = kLoraPieces<W> - 1; g >= 0; --g)
#pragma unroll
                        for (int b = 0; b < NR; ++b) acc[t][b] = lora_mfma(W{}, w[b], P[g], acc[t][b]);
                }
            }
        } else {
            lf4 x[H][2];
#pragma unroll
            for (int t = 0; t < H; ++t)
                if (t == 0 || second) turn_rows128(lx, in.x[t], x[t]);
#pragma unroll
            for (int b = 0; b < NR; ++b) {
                lf4 w[2];
                turn_rows128(la, in.a[b], w);
#pragma unroll
                for (int t = 0; t < H; ++t) {
                    if (t > 0 && !second) continue;
#pragma unroll
                    for (int c = 0; c < 8; ++c)
                        acc[t][b] = __builtin_amdgcn_mfma_f32_16x16x4f32(w[c >> 2][c & 3], x[t][c >> 2][c & 3], acc[t][b], 0, 0, 0);
                }
            }
        }
    }
    // rk: the adapter's own rank
    __device__ inline void run(int rk) {
        const int wave = (int)threadIdx.x >> 6;
#pragma unroll
        for (int t = 0; t < H; ++t)
#pragma unroll
            for (int b = 0; b < NR; ++b) acc[t][b] = lf4{0, 0, 0, 0};
        In in[U];
        for (int s = s0 + wave; s < steps; s += U * NW) {
#pragma unroll
            for (int u = 0; u < U; ++u) load(in[u], min(s + u * NW, steps - 1));
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (s + u * NW < steps) mul(in[u]);
        }
        if (rest_is(wave)) {
            load_rest(in[0], steps);
            mul(in[0]);
        }
        if constexpr (kLoraPieces<W> > 0) {
            uint32_t most = 0;
#pragma unroll
            for (int t = 0; t < H; ++t)
#pragma unroll
                for (int b = 0; b < NR; ++b) most = max(most, largest(acc[t][b], 16 * b, rk));
            if (__builtin_expect(__any(most > kInfinity), 0)) again(wave, rk);
        }
    }
    // rare: the sums that are NaN once more in the f32 form, sixteen ranks of sixteen rows at a time (in few registers): always
    // the first ones, and the others move up
    __device__ inline void again(int wave, int rk) {
        constexpr int N = 8;
        const int end = steps + (rest_is(wave) ? 1 : 0);
#pragma unroll 1
        for (int j = 0; j < H * NR; ++j) {
            const bool bad = __any(largest(acc[0][0], 16 * (j % NR), rk) > kInfinity);
            const float* row[2] = {j < NR ? xr[0][0] : xr[H - 1][0], j < NR ? xr[0][1] : xr[H - 1][1]};
            const typename W::T* w0 = A + (uint32_t)min(16 * (j % NR) + a_row(0), rank - 1) * (uint32_t)k;
            lf4 sum = {0, 0, 0, 0};
            for (int s = s0 + wave; bad && s < end; s += NW) {
                const int c0 = s * 32 + 4 * (lane & 7), i0 = s * 32 + a_col();
                lf4 in[2], x[2];
                union {
                    typename W::T t[N];
                    lf4 v;
                } a;
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int c = 0; c < 4; ++c) in[h][c] = c0 + c < k ? row[h][c0 + c] : 0.0f;
#pragma unroll
                for (int c = 0; c < N; ++c) a.t[c] = i0 + c < k ? w0[i0 + c] : (typename W::T)0;
                turn_rows128(lx, in, x);
                const LoraWords w = __builtin_bit_cast(LoraWords, turn_rows64(la, a.v));
#pragma unroll
                for (int c = 0; c < 8; ++c)
                    sum = __builtin_amdgcn_mfma_f32_16x16x4f32(lora_value<W>(w, c), x[c >> 2][c & 3], sum, 0, 0, 0);
            }
            lf4 done;
#pragma unroll
            for (int i = 0; i < 4; ++i) done[i] = bad && acc[0][0][i] != acc[0][0][i] ? sum[i] : acc[0][0][i];
#pragma unroll
            for (int b = 0; b < H * NR; ++b) acc[b / NR][b % NR] = b + 1 < H * NR ? acc[(b + 1) / NR % H][(b + 1) % NR] : done;
        }
    }
    // the largest magnitude's word, times two, of sums below the adapter's own rank; above kInfinity it is a NaN
    static constexpr uint32_t kInfinity = 0xFF000000u;
    __device__ inline uint32_t largest(const lf4& sums, int r0, int rk) const {
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) m = max(m, (2u * __float_as_uint(sums[i])) & (uint32_t)((r0 + 4 * q + i - rk) >> 31));
        return m;
    }
    // part as above, of sixteen t of the tile
    __device__ inline void give(float* part, int t) const {
        const int wave = (int)threadIdx.x >> 6;
        float* mine = part + (size_t)wave * 16 * NR * kLoraPart;
#pragma unroll
        for (int h = 0; h < H; ++h) {
            if (h != t) continue;
#pragma unroll
            for (int b = 0; b < NR; ++b)
#pragma unroll
                for (int i = 0; i < 4; ++i) mine[(16 * b + 4 * q + i) * kLoraPart + p] = acc[h][b][i];
        }
    }
    // k's rest belongs to the wave whose turn it is after the last whole step of all
    __device__ inline bool rest_is(int wave) const {
        return steps == k / 32 && k % 32 != 0 && (steps - s0) % NW == wave;
    }
};

// y = base + S B^T over columns c0 .. c1 of the tile, in steps of 64 columns per wave: product j of four has the
// columns o0 + 4 n + j, so that a lane holds four neighbouring columns (4 (lane % 16)) of each
// of the rows 4 (lane / 16) .. +3, and a load or store covers 256 bytes of four rows.
// The ranks of a lane's 4 NR values of a row of B and of S: groups of GW from 4 NR (lane / 16) on; a
// group that reaches past the rank is moved back to the row's last GW (rows of fewer than four: the
// last value again), so that loads stay inside the row.  A value counts if it is not one that an
// earlier group has, and below the adapter's own rank; the others' weights become zeros by a
// mask in registers (a NaN or an infinity past an adapter's own rank must not meet its zero in S).
template <int NR>
constexpr int kLoraGroupWidth = NR == 1 ? 4 : 8;
// the rank of value j of a row's 16 NR (lane j / (4 NR)'s j % (4 NR)), and whether it counts
template <int NR>
__device__ inline int lora_value_at(int j, int rank) {
    constexpr int GW = kLoraGroupWidth<NR>;
    return min(j / GW * GW, max(0, rank - GW)) + j % GW;
}
template <int NR>
__device__ inline bool lora_value_counts(int j, int rank, int rk) {
    const int r = lora_value_at<NR>(j, rank);
    return r >= j / kLoraGroupWidth<NR> * kLoraGroupWidth<NR> && r < rk;
}
template <typename W, int NR, int NW, int H, bool STREAM>
struct LoraExpand {
    static constexpr int GW = kLoraGroupWidth<NR>, NG = 4 * NR / GW;
    typedef typename std::conditional<NR == 1, typename W::V4, typename W::V8>::type V;
    const typename W::T* B;                                 // rows * rank is below 2^28
    const uint8_t* base[H][4];                              // of the lane's four rows of each sixteen; null: zeros
    uint8_t* dst[H][4];
    int rank, rows, c1, n, p, q, at[NG];
    bool based;

    // row: of the lane's places lane % 16 in the tile of n rows
    __device__ inline LoraExpand(const LoraArgs& a, const typename W::T* B_, const int (&row)[H], int n_, int c1_)
        : B(B_), rank(a.rank), rows(a.rows), c1(c1_), n(n_), based(a.base != nullptr) {
        const int lane = (int)threadIdx.x & 63;
        p = lane & 15;
        q = lane >> 4;
#pragma unroll
        for (int h = 0; h < H; ++h)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int r = __shfl(row[h], 4 * q + i);
                base[h][i] = a.base ? a.base + lora_at(r, a.n_ids, a.base_id, a.base_tok) : nullptr;
                dst[h][i] = a.dst + lora_at(r, a.n_ids, a.dst_id, a.dst_tok);
            }
#pragma unroll
        for (int g = 0; g < NG; ++g) at[g] = min(4 * NR * q + GW * g, max(0, rank - GW));
    }
    // all bits of a value that counts, else none: by the signs, since conditions for every value fill the scalar registers
    __device__ inline uint32_t counts(int j, int rk) const {
        const int r = at[j / GW] + j % GW;
        return ~(uint32_t)(((r - (4 * NR * q + j / GW * GW)) | (rk - 1 - r)) >> 31);
    }
    __device__ inline void load_w(V (&w)[4][NG], int o0) const {
#pragma unroll
        for (int h = 0; h < 4; ++h) {
            const typename W::T* row = B + (uint32_t)min(o0 + 4 * p + h, rows - 1) * (uint32_t)rank;
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                if constexpr (NR == 1) {
                    if (rank < 4) {
#pragma unroll
                        for (int c = 0; c < 4; ++c) W::set(w[h][g], c, row[min(c, rank - 1)]);
                    } else {
                        w[h][g] = W::load4(row + at[g]);
                    }
                } else {
                    w[h][g] = W::load8(row + at[g]);
                }
            }
        }
    }
    __device__ inline void load_y(lf4 (&y)[4], int t, int o0) const {
        const int o = o0 + 4 * p;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            y[i] = lf4{0, 0, 0, 0};
            if (!based) continue;
            const float* b = reinterpret_cast<const float*>(base[t][i]) + o;
            if (o + 4 <= c1) {
                y[i] = *reinterpret_cast<const lf4u*>(b);
            } else {
#pragma unroll
                for (int c = 0; c < 4; ++c)
                    if (o + c < c1) y[i][c] = b[c];
            }
        }
    }
    // Streamed past the caches in large calls: their output does not fit there, and A and B, which the other tiles read again,
    // stay (16,384 rows at rank 32: 95 us against 99, and 82 against 97 where x and base come from the last-level cache)
    __device__ inline void store(const lf4 (&in)[4], const lf4 (&d)[4], int t, int o0, unsigned rows_in) const {
        const int o = o0 + 4 * p;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (!((rows_in >> (4 * q + i)) & 1u)) continue;
            lf4 y;
#pragma unroll
            for (int j = 0; j < 4; ++j) y[j] = in[i][j] + d[j][i];
            float* b = reinterpret_cast<float*>(dst[t][i]) + o;
            if (o + 4 <= c1) {
                if constexpr (STREAM) __builtin_nontemporal_store(y, reinterpret_cast<lf4u*>(b));
                else *reinterpret_cast<lf4u*>(b) = y;
            } else {
#pragma unroll
                for (int c = 0; c < 4; ++c)
                    if (o + c < c1) b[c] = y[c];
            }
        }
    }
    // The wave's steps from o0 on.  s: the lane's S, already scaled, zeros where a value does not count
    __device__ inline void run(int o0, const float (&s)[H][4 * NR], int rk) const {
        constexpr int NP = (NR + 1) / 2, N = kLoraPieces<W>, M = N > 0 ? 2 : 1;   // products of 32 ranks, pieces, values of a mask
        uint32_t mask[4 * NR / M];
#pragma unroll
        for (int j = 0; j < 4 * NR / M; ++j) {
            if constexpr (M == 2) mask[j] = (counts(2 * j, rk) & 0xFFFFu) | (counts(2 * j + 1, rk) & 0xFFFF0000u);
            else mask[j] = counts(j, rk);
            asm volatile("" : "+v"(mask[j]));               // kept as a word
        }
        // the rows to be written, and of them those with values too small for f16 pieces
        unsigned rows_in[H], alone[H];
        LoraWords P[H][NP][N > 0 ? N : 1];
        float back[H][4];                                   // of the lane's four rows
#pragma unroll
        for (int t = 0; t < H; ++t) {
            rows_in[t] = (unsigned)((1u << max(0, min(16, n - 16 * t))) - 1u);
            alone[t] = 0u;
#pragma unroll
            for (int i = 0; i < 4; ++i) back[t][i] = 1.0f;
            if constexpr (N > 0) {
                const float most = lora_most(s[t], 0.0f);
                float scale = 1.0f;
                bool some = false;
                if constexpr (std::is_same<W, LoraF16>::value) {
                    float mine;
                    scale = lora_scale_of(lora_column_most(most), mine);
#pragma unroll
                    for (int i = 0; i < 4; ++i) back[t][i] = __shfl(mine, 4 * q + i);
                }
#pragma unroll
                for (int b = 0; b < NP; ++b) {
                    float v[8];
#pragma unroll
                    for (int c = 0; c < 8; ++c) v[c] = 8 * b + c < 4 * NR ? s[t][(8 * b + c) % (4 * NR)] : 0.0f;
                    if constexpr (std::is_same<W, LoraF16>::value) some |= lora_split(W{}, v, scale, P[t][b]);
                    else lora_split(W{}, v, scale, P[t][b]);
                }
                if (__any(some)) alone[t] = lora_rows_of(__ballot(some)) & rows_in[t];
            }
        }
        for (; o0 < c1; o0 += 64 * NW) {
            V w[4][NG];
            lf4 y[H][4];
#pragma unroll
            for (int t = 0; t < H; ++t)
                if (t == 0 || n > 16 * t) load_y(y[t], t, o0);
            load_w(w, o0);
            LoraWords ww[NP][4];                            // 16-bit weights: the operands
            if constexpr (N > 0) {
#pragma unroll
                for (int b = 0; b < NP; ++b)
#pragma unroll
                    for (int h = 0; h < 4; ++h) {
                        if constexpr (NR == 1) {
                            const uint2 r = __builtin_bit_cast(uint2, w[h][0]);
                            ww[b][h] = LoraWords{{r.x, r.y, 0, 0}};
                        } else {
                            ww[b][h] = __builtin_bit_cast(LoraWords, w[h][b]);
                        }
#pragma unroll
                        for (int c = 0; c < 4; ++c)
                            if (4 * b + c < 2 * NR) ww[b][h].u[c] &= mask[(4 * b + c) % (4 * NR / M)];
                    }
            }
#pragma unroll
            for (int t = 0; t < H; ++t) {
                if (t > 0 && n <= 16 * t) continue;
                lf4 d[4] = {{0, 0, 0, 0}, {0, 0, 0, 0}, {0, 0, 0, 0}, {0, 0, 0, 0}};
                if constexpr (N > 0) {
#pragma unroll
                    for (int b = 0; b < NP; ++b)
#pragma unroll
                        for (int g = N - 1; g >= 0; --g)
#pragma unroll
                            for (int h = 0; h < 4; ++h) d[h] = lora_mfma(W{}, P[t][b][g], ww[b][h], d[h]);
                    if constexpr (std::is_same<W, LoraF16>::value) {
#pragma unroll
                        for (int h = 0; h < 4; ++h)
#pragma unroll
                            for (int i = 0; i < 4; ++i) d[h][i] *= back[t][i];
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < 4 * NR; ++j)
#pragma unroll
                        for (int h = 0; h < 4; ++h) {
                            const float v = __uint_as_float(__float_as_uint(W::get(w[h][j / GW], j % GW)) & mask[j % (4 * NR / M)]);
                            d[h] = __builtin_amdgcn_mfma_f32_16x16x4f32(s[t][j], v, d[h], 0, 0, 0);
                        }
                }
                unsigned apart = 0u;                        // rare: rows in the f32 form
                if constexpr (N > 0) {
                    apart = alone[t];
                    bool nan[4], any = false;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        nan[i] = __builtin_isunordered(d[0][i], d[1][i]) || __builtin_isunordered(d[2][i], d[3][i]);
                        any |= nan[i];
                    }
                    if (__builtin_expect(__any(any), 0)) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const uint64_t m = __ballot(nan[i]);
#pragma unroll
                            for (int r = 0; r < 4; ++r) apart |= ((m >> (16 * r)) & 0xFFFFu ? 1u : 0u) << (4 * r + i);
                        }
                        apart &= rows_in[t];
                    }
                }
                store(y[t], d, t, o0, rows_in[t] & ~apart);
                if constexpr (N > 0) {
                    if (__builtin_expect(apart != 0u, 0)) {
                        lf4 e[4] = {{0, 0, 0, 0}, {0, 0, 0, 0}, {0, 0, 0, 0}, {0, 0, 0, 0}};
#pragma unroll
                        for (int j = 0; j < 4 * NR; ++j)
#pragma unroll
                            for (int h = 0; h < 4; ++h)
                                e[h] = __builtin_amdgcn_mfma_f32_16x16x4f32(s[t][j], lora_value<W>(ww[j / 8][h], j % 8), e[h], 0, 0, 0);
                        store(y[t], e, t, o0, apart);
                    }
                }
            }
        }
    }
};

// the lane's operand of S^T, of row lane % 16, times c; 0 where a value does not count
template <int NR, int NW, typename E_>
__device__ inline void lora_sum_parts(const E_& E, const float* part, int rk, float c, float (&s)[4 * NR]) {
    constexpr int GW = E_::GW;
#pragma unroll
    for (int j = 0; j < 4 * NR; ++j) {
        const int r = E.at[j / GW] + j % GW;
        float v = 0.0f;
#pragma unroll
        for (int w = 0; w < NW; ++w) v += part[((size_t)w * 16 * NR + r) * kLoraPart + E.p];
        s[j] = __uint_as_float(__float_as_uint(v * c) & E.counts(j, rk));
    }
}

template <typename W>
__device__ inline const typename W::T* lora_a(const LoraArgs& a, int key) {
    return static_cast<const typename W::T*>(a.a) + (size_t)key * a.rank * a.k;
}
template <typename W>
__device__ inline const typename W::T* lora_b(const LoraArgs& a, int key) {
    return static_cast<const typename W::T*>(a.b) + (size_t)key * a.rows * a.rank;
}

// The shrink and the expand of a tile in one workgroup, for the calls at both ends (between them the two
// kernels below).  Small ones, in one launch: a workgroup finds its tile by itself (FIND)
// and shrinks it whole, also when several share its columns; up to U steps of loads at a time, which it
// waits for.  Large ones, with tiles to fill the chip, take them from the lists, and hold OCC
// waves per SIMD to cover the loads.  Bound by HBM there: 16,384 rows, 2048 x 2048, rank 32, 402 MB in 95 us (4.2 TB/s; a
// large copy reaches 4.7).  One token: 7.5 us, of which the smallest launch takes 3.6; loads of B and base under the shrink
// made it no shorter.  grid (slots, column parts, windows).
template <typename W, int NR, int NW, int U, int OCC, bool FIND>
__global__ __launch_bounds__(64 * NW, OCC) void k_lora_apply(LoraArgs a, LoraTiles t) {
    __shared__ float part[NW * 16 * NR * kLoraPart];
    __shared__ lf4 turn[NW * (kLoraXLds + kLoraALds<W>)];
    __shared__ typename std::conditional<FIND, LoraFind<NW>, int>::type find;
    int key, n, row[1], pos;
    if constexpr (FIND) {
        if (!lora_tile<NW>(a, t, find, key, n, row)) return;
    } else {
        if (!lora_item(t, (int)blockIdx.z, key, n, row, pos)) return;
    }
    const int c0 = (int)blockIdx.y * t.cols, c1 = min(a.rows, c0 + t.cols), o0 = c0 + 64 * ((int)threadIdx.x >> 6);
    if (key < 0) {
        lora_plain_rows(a, key, n, row, c0, c1);
        return;
    }
    const int rk = lora_rank(a, key);
    const float c = lora_scale(a, key);
    LoraShrink<W, NR, NW, U, 1> S(a, lora_a<W>(a, key), row, n, turn, 0, 1 << 28);
    S.run(rk);
    const LoraExpand<W, NR, NW, 1, !FIND> E(a, lora_b<W>(a, key), row, n, c1);
    float s[1][4 * NR];
    S.give(part, 0);
    __syncthreads();
    lora_sum_parts<NR, NW>(E, part, rk, c, s[0]);
    E.run(o0, s, rk);
}

// Larger calls: S = X A^T of a tile and one part of k per workgroup, to t.s, [k parts][position in order][16 NR]
// in all, a tile of n rows as the expand reads it: [4 NR groups of four values][n rows][4] of every lane's values in
// lora_value_at's order (zeros where one does not count), so that its loads are whole lines.  grid (slots, k parts, windows).
template <typename W, int NR, int NW, int U, int H, bool HALF>
__device__ inline void lora_shrink_part(const LoraArgs& a, const LoraTiles& t, int w, float* part, lf4* turn) {
    int key, n, row[H], pos;
    const int part_k = HALF ? 0 : (int)blockIdx.y, h0 = HALF ? 16 * (int)blockIdx.y : 0;
    if (part_k >= t.k_parts || !lora_item(t, w, key, n, row, pos, h0) || key < 0) return;
    const int s0 = part_k * t.k_steps, rk = lora_rank(a, key);
    constexpr int ROWS = HALF ? 32 : 16 * H;                // of the tile
    LoraShrink<W, NR, NW, U, H> S(a, lora_a<W>(a, key), row, n, turn, s0, s0 + t.k_steps);
    S.run(rk);
    float* out = t.s + ((size_t)part_k * t.positions + pos) * (16 * NR);
    const size_t slot = (size_t)w * t.slots + blockIdx.x;
    const float c = t.scaled ? lora_scale(a, key) : 1.0f;
#pragma unroll
    for (int h = 0; h < H; ++h) {
        if (h) __syncthreads();
        S.give(part, h);
        __syncthreads();
        const int g = h0 + 16 * h, m = n - g;                // rows of this sixteen: part holds the last one's again past them
        if (m > 0)
            for (int i = (int)threadIdx.x; i < 16 * 16 * NR; i += 64 * NW) {
                const int j = i / 16, p = i % 16, r = lora_value_at<NR>(j, a.rank);     // value j of the 16 NR, row p
                float v = 0.0f;
#pragma unroll
                for (int w4 = 0; w4 < NW; ++w4) v += part[(w4 * 16 * NR + r) * kLoraPart + p];
                if (p < m) out[((j >> 2) * n + g + p) * 4 + (j & 3)] = lora_value_counts<NR>(j, a.rank, rk) ? v : 0.0f;
            }
        if (!t.pieces) continue;
        // As the weights' gradients read it: in bf16 pieces, a rank's rows side by side, zeros past the tile's rows and the
        // adapter's rank; and where the rows of x are (past the last row, the last)
        if (threadIdx.x < 16) {
            const int tok = row[h] / a.n_ids;
            t.off[slot * ROWS + g + threadIdx.x] =
                (uint64_t)tok * a.x_tok + (uint64_t)((row[h] - tok * a.n_ids) % a.x_rows) * a.x_id;
        }
        for (int i = (int)threadIdx.x; i < 16 * 8 * NR; i += 64 * NW) {
            const int r = i / 8, p = 2 * (i % 8);           // two rows at a time
            float v[2] = {0.0f, 0.0f};
#pragma unroll
            for (int e = 0; e < 2; ++e)
                if (p + e < m && r < rk) {
#pragma unroll
                    for (int w4 = 0; w4 < NW; ++w4) v[e] += part[(w4 * 16 * NR + r) * kLoraPart + p + e];
                    v[e] *= c;
                }
#pragma unroll
            for (int z = 0; z < 3; ++z)
                reinterpret_cast<uint32_t*>(t.pieces)[((slot * 3 + z) * (16 * NR) + r) * (ROWS / 2) + g / 2 + i % 8] = lora_split2(v);
        }
    }
}
// Both sides' in one launch, the windows of the second after the first's (forward: windows of b none)
template <typename W, int NR, int NW, int U, int OCC, int H, bool HALF>
__global__ __launch_bounds__(64 * NW, OCC) void k_lora_shrink(LoraArgs a, LoraTiles t, LoraArgs b, LoraTiles u, int windows) {
    __shared__ float part[NW * 16 * NR * kLoraPart];
    __shared__ lf4 turn[NW * (kLoraXLds + kLoraALds<W>)];
    const int w = (int)blockIdx.z;
    if (w < windows) lora_shrink_part<W, NR, NW, U, H, HALF>(a, t, w, part, turn);
    else lora_shrink_part<W, NR, NW, U, H, HALF>(b, u, w - windows, part, turn);
}

// y = base + c S B^T of a tile and t.cols columns.  grid (slots, column parts, windows).
template <typename W, int NR, int OCC, int H>
__global__ __launch_bounds__(256, OCC) void k_lora_expand(LoraArgs a, LoraTiles t) {
    constexpr int NW = 4;
    int key, n, row[H], pos;
    if (!lora_item(t, (int)blockIdx.z, key, n, row, pos)) return;
    const int c0 = (int)blockIdx.y * t.cols, c1 = min(a.rows, c0 + t.cols), o0 = c0 + 64 * ((int)threadIdx.x >> 6);
    if (key < 0) {
        lora_plain_rows(a, key, n, row, c0, c1);
        return;
    }
    if (o0 >= c1) return;
    const int rk = lora_rank(a, key);
    const float c = lora_scale(a, key);
    const LoraExpand<W, NR, NW, H, true> E(a, lora_b<W>(a, key), row, n, c1);
    float s[H][4 * NR];
#pragma unroll
    for (int h = 0; h < H; ++h) {
        const float* in = t.s + (size_t)pos * (16 * NR) + (NR * E.q * n + min(16 * h + E.p, n - 1)) * 4;
        lf4 v[NR];
#pragma unroll
        for (int j = 0; j < NR; ++j) v[j] = lf4{0, 0, 0, 0};
        constexpr int Z = NR == 8 ? 1 : 4;                  // the parts in order, the loads of Z at a time
        for (int z = 0; z < t.k_parts; z += Z) {
            lf4 l[Z][NR];
#pragma unroll
            for (int y = 0; y < Z; ++y) {
                if (z + y >= t.k_parts) continue;
#pragma unroll
                for (int j = 0; j < NR; ++j)
                    l[y][j] = *reinterpret_cast<const lf4*>(in + (size_t)(z + y) * t.positions * (16 * NR) + j * n * 4);
            }
#pragma unroll
            for (int y = 0; y < Z; ++y)
                if (z + y < t.k_parts) {
#pragma unroll
                    for (int j = 0; j < NR; ++j) v[j] += l[y][j];
                }
        }
#pragma unroll
        for (int j = 0; j < 4 * NR; ++j) s[h][j] = v[j / 4][j % 4] * c;
    }
    E.run(o0, s, rk);
}

// ---------------------------------------------------------------------------
// Backward.  s = A x and u = c B^T dy of every row are shrinks (of x by A, of dy by B^T) and dx = A^T u is an
// expand, on transposed copies of the pairs in use; dA = sum u x^T and dB = c sum dy s^T are sums over a key's rows.
// ---------------------------------------------------------------------------

// whether any window has rows of the key; the whole workgroup asks
__device__ inline bool lora_key_used(const uint32_t* runs, int windows, int keys, int key) {
    uint32_t any = 0;
    for (int w = (int)threadIdx.x; w < windows; w += (int)blockDim.x) any |= runs[(size_t)w * keys + key];
    return __syncthreads_or(any != 0u);
}

struct LoraTurn {
    const void *a, *b;            // [keys][rank][k], [keys][rows][rank]
    void *at, *bt;                // [keys][k][rank], [keys][rank][rows]
    const uint32_t* runs;
    int windows, keys, rank, k, rows, tiles_a;
};
// 64 columns of A, or rows of B, per workgroup, through LDS: both sides are read and written along their rows.
// grid (64s of k, then of rows; keys)
template <typename T>
__global__ __launch_bounds__(256) void k_lora_transpose(LoraTurn a) {
    __shared__ T s[64 * (kLoraMaxRank + 2)];
    const int key = (int)blockIdx.y, rank = a.rank, pitch = rank + 2;
    if (!lora_key_used(a.runs, a.windows, a.keys, key)) return;
    const bool of_a = (int)blockIdx.x < a.tiles_a;
    const int n = of_a ? a.k : a.rows, c0 = 64 * ((int)blockIdx.x - (of_a ? 0 : a.tiles_a)), m = min(64, n - c0);
    const T* in = static_cast<const T*>(of_a ? a.a : a.b) + (size_t)key * rank * n;
    T* out = static_cast<T*>(of_a ? a.at : a.bt) + (size_t)key * rank * n;
    // i / rank for i below 64 * rank, exactly: the reciprocal is too large by less than 2^-20, i below 2^13
    const uint32_t inv = ((1u << 20) + rank - 1) / rank;
    auto over = [&](int i) { return (int)(((uint32_t)i * inv) >> 20); };
    constexpr int U = 8;                                    // loads at a time
    for (int i0 = (int)threadIdx.x; i0 < 64 * rank; i0 += 256 * U) {
        T v[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = min(i0 + 256 * u, 64 * rank - 1), j = over(i), c = min(of_a ? i & 63 : j, m - 1), r = of_a ? i >> 6 : i - j * rank;
            v[u] = in[of_a ? (size_t)r * n + c0 + c : (size_t)(c0 + c) * rank + r];
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = i0 + 256 * u, j = over(min(i, 64 * rank - 1));
            if (i < 64 * rank) s[(of_a ? i & 63 : j) * pitch + (of_a ? i >> 6 : i - j * rank)] = v[u];
        }
    }
    __syncthreads();
#pragma unroll 4
    for (int i = (int)threadIdx.x; i < 64 * rank; i += 256) {
        const int j = over(i), c = of_a ? j : i & 63, r = of_a ? i - j * rank : i >> 6;
        if (c < m) out[of_a ? (size_t)(c0 + c) * rank + r : (size_t)r * n + c0 + c] = s[c * pitch + r];
    }
}

struct LoraGrad {
    const uint32_t* runs;
    int windows, keys, slots, splits, rank;
    int tiles_a;                  // column tiles of dA; dB's follow
    const uint16_t* p[2];         // pieces of u, of s (tiles of 32 rows)
    const uint64_t* off[2];       // offsets of x's rows, of dy's
    const uint8_t* src[2];        // x, dy
    int width[2];                 // k, rows
    float* out[2];                // dA, dB
    float* part[2];               // several splits: [splits][keys][tiles][16 NR][64]; window w is split w % splits'
    const float* scale;
    const int32_t* ranks;
    int n_experts, add;
};

// 16 ranks (rank block b) by 64 columns, summed in sum[16][64] of LDS, to the gradient.  dA [rank][k], dB [rows][rank].
// Past the adapter's own rank the pieces are zeros, but 0 times an infinity of x or dy is not.
__device__ inline void lora_grad_store(const LoraGrad& g, int side, int key, int b, int c0, const float* sum) {
    const int tid = (int)threadIdx.x, n = g.width[side];
    float* out = g.out[side] + (size_t)key * g.rank * n;
    const float c = side && g.scale ? g.scale[key / g.n_experts] : 1.0f;
    const int rk = g.ranks ? g.ranks[key / g.n_experts] : g.rank;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int e = tid + 256 * i, r = side ? e & 15 : e >> 6, o = side ? e >> 4 : e & 63;
        if (16 * b + r >= g.rank || c0 + o >= n) continue;
        float* to = out + (side ? (size_t)(c0 + o) * g.rank + 16 * b + r : (size_t)(16 * b + r) * n + c0 + o);
        const bool in = 16 * b + r < rk;
        const float v = in ? sum[r * 64 + o] * c : 0.0f;
        if (!g.add) *to = v;
        else if (in) *to = *to + v;
    }
}

// The splits that have rows of the key, a bit each (at most 32); a wave asks.  first: the lane's run of the first 64 windows
__device__ inline uint32_t lora_grad_splits(const LoraGrad& g, int key, uint32_t& first) {
    const int lane = (int)threadIdx.x & 63;
    uint32_t used = 0;
    first = 0;
    for (int w = lane; w < g.windows; w += 64) {
        const uint32_t r = g.runs[(size_t)w * g.keys + key];
        if (w == lane) first = r;
        used |= (r != 0u ? 1u : 0u) << (w % g.splits);
    }
    uint32_t all = 0;
    for (int z = 0; z < g.splits; ++z) all |= (__ballot((used >> z) & 1u) ? 1u : 0u) << z;
    return all;
}

// dA or dB of one key and 64 columns: rank blocks of 16 by columns, summed over the key's tiles, 32 rows and one
// v_mfma_f32_16x16x32_bf16 each, which the waves share.  Both operands are f32 in three bf16 pieces; the six
// products above 2^-24 of the whole are kept: 96 cycles where the f32 form takes 256.  Column 4 n + j
// of x (dy) belongs to product j of four, so a lane loads four neighbours of eight rows, 256 bytes
// a row; the next tiles' rows are loaded under the products.  splits > 1: a workgroup takes
// the windows of its split, and if others have rows of the key too k_lora_grad_sum adds them up.
// grid (column tiles, keys, splits)
template <int NR, int OCC>
__global__ __launch_bounds__(256, OCC) void k_lora_grad(LoraGrad g) {
    constexpr int RB = NR < 4 ? NR : 4;                     // rank blocks summed at a time
    __shared__ float sum[4][RB * 16 * 64];
    const int lane = (int)threadIdx.x & 63, p = lane & 15, q = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int side = (int)blockIdx.x < g.tiles_a ? 0 : 1, tile = (int)blockIdx.x - (side ? g.tiles_a : 0), c0 = 64 * tile;
    const int key = (int)blockIdx.y, split = (int)blockIdx.z, n = g.width[side], col = c0 + 4 * p;
    uint32_t e;
    const uint32_t used = lora_grad_splits(g, key, e);
    // a key without rows: split 0 writes its zeros, but where they would be added (another call may be adding to that pair)
    if (!((used >> split) & 1u) && !(used == 0u && split == 0 && !g.add)) return;
    lf4 acc[NR][4];
#pragma unroll
    for (int b = 0; b < NR; ++b)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[b][j] = lf4{0, 0, 0, 0};
    // the key's tiles, every fourth this wave's, 64 windows at a time
    auto own = [&](int w) { return w < g.windows && w % g.splits == split; };
    int wb = 0, left = 0, turn = -1;
    uint64_t some = __ballot(e != 0u && own(lane));
    size_t at = 0;
    auto advance = [&](size_t& slot) {
        for (;;) {
            if (left > 0) {
                slot = at++;
                --left;
                turn = (turn + 1) & 3;
                if (turn == wave) return true;
                continue;
            }
            while (some == 0) {
                wb += 64;
                if (wb >= g.windows) return false;
                e = own(wb + lane) ? g.runs[(size_t)(wb + lane) * g.keys + key] : 0u;
                some = __ballot(e != 0u);
            }
            const int l = __builtin_ctzll(some);
            some &= some - 1ull;
            const uint32_t r = (uint32_t)__builtin_amdgcn_readlane((int)e, l);
            left = ((int)(r >> 16) + 31) / 32;
            at = (size_t)(wb + l) * g.slots + (r & 0xFFFFu);
        }
    };
    auto load_off = [&](uint64_t (&off)[8], size_t slot) {
        const uint64_t* o = g.off[side] + slot * 32 + 8 * q;
#pragma unroll
        for (int i = 0; i < 8; ++i) off[i] = o[i];
    };
    auto load_x = [&](lf4 (&x)[8], const uint64_t (&off)[8]) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float* row = reinterpret_cast<const float*>(g.src[side] + off[i]);
            if (col + 4 <= n) {
                x[i] = *reinterpret_cast<const lf4u*>(row + col);
            } else {
#pragma unroll
                for (int c = 0; c < 4; ++c) x[i][c] = col + c < n ? row[col + c] : 0.0f;
            }
        }
    };
    lf4 x[8];
    uint64_t off[8];
    size_t slot = 0, slot2 = 0;
    bool more = advance(slot);
    if (more) {
        load_off(off, slot);
        load_x(x, off);
    }
    while (more) {
        // this step's pieces and the next one's offsets; x to pieces; the next x, under the products
        more = advance(slot2);
        const uint16_t* pieces = g.p[side] + slot * (1536 * NR) + 32 * p + 8 * q;
        constexpr int UB = NR < 4 ? NR : 4;
        LoraWords U[UB][3];
#pragma unroll
        for (int b = 0; b < UB; ++b)
#pragma unroll
            for (int z = 0; z < 3; ++z) U[b][z] = *reinterpret_cast<const LoraWords*>(pieces + z * (512 * NR) + 512 * b);
        if (more) load_off(off, slot2);
        LoraWords X[4][3];
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                float v[2] = {x[2 * c][j], x[2 * c + 1][j]};
#pragma unroll
                for (int z = 0; z < 3; ++z) X[j][z].u[c] = lora_split2(v);
            }
        if (more) load_x(x, off);
#pragma unroll
        for (int b = 0; b < NR; ++b) {
            LoraWords V[3];
#pragma unroll
            for (int z = 0; z < 3; ++z) {
                V[z] = U[b % UB][z];
                if (b + UB < NR) U[b % UB][z] = *reinterpret_cast<const LoraWords*>(pieces + z * (512 * NR) + 512 * (b + UB));
            }
#pragma unroll
            for (int lo = 2; lo >= 0; --lo)                 // the smallest products first; four sums in turn
#pragma unroll
                for (int z = 0; z <= lo; ++z)
#pragma unroll
                    for (int j = 0; j < 4; ++j) acc[b][j] = lora_mfma(LoraBF16{}, V[z], X[j][lo - z], acc[b][j]);
        }
        slot = slot2;
    }
    const bool whole = (used & (used - 1u)) == 0u;          // no other split has rows
#pragma unroll
    for (int b0 = 0; b0 < NR; b0 += RB) {
        if (16 * b0 >= g.rank) break;
        if (b0) __syncthreads();
#pragma unroll
        for (int b = 0; b < RB; ++b)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                *reinterpret_cast<lf4*>(&sum[wave][b * 1024 + (4 * q + i) * 64 + 4 * p]) =
                    lf4{acc[b0 + b][0][i], acc[b0 + b][1][i], acc[b0 + b][2][i], acc[b0 + b][3][i]};
        __syncthreads();
        lf4* to = reinterpret_cast<lf4*>(sum[0]);
        if (!whole) to = reinterpret_cast<lf4*>(g.part[side] + ((((size_t)split * g.keys + key) * ((n + 63) / 64) + tile) * NR + b0) * (16 * 64));
#pragma unroll
        for (int b = 0; b < RB; ++b) {
            const int o = (int)threadIdx.x + 256 * b;
            lf4 v = reinterpret_cast<const lf4*>(sum[0])[o];
#pragma unroll
            for (int w = 1; w < 4; ++w) v += reinterpret_cast<const lf4*>(sum[w])[o];
            to[o] = v;
        }
        if (whole) {
            __syncthreads();
            for (int b = 0; b < RB && 16 * (b0 + b) < g.rank; ++b) lora_grad_store(g, side, key, b0 + b, c0, sum[0] + 1024 * b);
        }
    }
}

// grid (column tiles, keys, blocks of 16 ranks)
template <int NR>
__global__ __launch_bounds__(256) void k_lora_grad_sum(LoraGrad g) {
    __shared__ float sum[16 * 64];
    const int side = (int)blockIdx.x < g.tiles_a ? 0 : 1, tile = (int)blockIdx.x - (side ? g.tiles_a : 0);
    const int key = (int)blockIdx.y, b = (int)blockIdx.z, tiles = (g.width[side] + 63) / 64;
    uint32_t e;
    const uint32_t used = lora_grad_splits(g, key, e);
    if ((used & (used - 1u)) == 0u) return;                 // written by its only split
    lf4 v = {0, 0, 0, 0};
    for (uint32_t left = used; left; left &= left - 1u)
        v += reinterpret_cast<const lf4*>(g.part[side] + ((((size_t)__builtin_ctz(left) * g.keys + key) * tiles + tile) * NR + b) * (16 * 64))[threadIdx.x];
    reinterpret_cast<lf4*>(sum)[threadIdx.x] = v;
    __syncthreads();
    lora_grad_store(g, side, key, b, 64 * tile, sum);
}

}  // namespace sabah
