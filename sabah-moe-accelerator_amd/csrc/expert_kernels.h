// Products of experts kept in float types (f32, f16, bf16), grouped by expert with ragged sizes, and
// their gradients.  Row r = t * n_ids + i is (token t, slot i); e_r = ids[t][i], -1: none.
//   forward    y_r = W[e_r] x_r
//   backward   dx_r = W[e_r]^T dy_r;   dW[e] (+)= sum over the rows of e of dy_r x_r^T
// Products are exact in f32, sums are f32 on the matrix cores; y and dx are rounded once, dW is f32.
//
// k_expert_count, _scan, _place: the rows in expert order, stable and without an order that depends on
//   atomics, so the same ids give the same bits; cut into tiles of one expert.
// k_expert_gemm:  a tile of 128 rows by 128 columns, both operands staged through LDS.
// k_expert_rows:  up to 16 rows of one expert (decode, few tokens): W streamed from HBM into MFMA operands.
#pragma once
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

namespace sabah {

// ---------------------------------------------------------------------------
// storage types
// ---------------------------------------------------------------------------
typedef float xf4 __attribute__((ext_vector_type(4)));
typedef float xf16 __attribute__((ext_vector_type(16)));
typedef uint32_t xu4 __attribute__((ext_vector_type(4)));
typedef uint32_t xu2 __attribute__((ext_vector_type(2)));
typedef xu4 xu4u __attribute__((aligned(2)));   // one load or store at any address of the element's alignment
typedef xu2 xu2u __attribute__((aligned(2)));
typedef __bf16 xb8 __attribute__((ext_vector_type(8)));
typedef _Float16 xh8 __attribute__((ext_vector_type(8)));
typedef short xs4 __attribute__((ext_vector_type(4)));

// 16 bytes of an operand (8 values of 16 bits, 4 of 32) are summed over by one step: the lanes' halves (32x32) or
// quarters (16x16) hold neighbouring 16 bytes of both operands.
struct ExpF32 {
    typedef float S;
    static constexpr int kVec = 4;
    static __device__ inline xf16 mma32(xu4 a, xu4 b, xf16 c) {
        const xf4 x = __builtin_bit_cast(xf4, a), y = __builtin_bit_cast(xf4, b);
#pragma unroll
        for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_32x32x2f32(x[j], y[j], c, 0, 0, 0);
        return c;
    }
    static __device__ inline xf4 mma16(xu4 a, xu4 b, xf4 c) {
        const xf4 x = __builtin_bit_cast(xf4, a), y = __builtin_bit_cast(xf4, b);
#pragma unroll
        for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(x[j], y[j], c, 0, 0, 0);
        return c;
    }
    static __device__ inline S put(float v) { return v; }
};
struct ExpF16 {
    typedef _Float16 S;
    static constexpr int kVec = 8;
    static __device__ inline xf16 mma32(xu4 a, xu4 b, xf16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(xh8, a), __builtin_bit_cast(xh8, b), c, 0, 0, 0);
    }
    static __device__ inline xf4 mma16(xu4 a, xu4 b, xf4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(xh8, a), __builtin_bit_cast(xh8, b), c, 0, 0, 0);
    }
    static __device__ inline S put(float v) { return (_Float16)v; }
};
struct ExpBF16 {
    typedef __bf16 S;
    static constexpr int kVec = 8;
    static __device__ inline xf16 mma32(xu4 a, xu4 b, xf16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(xb8, a), __builtin_bit_cast(xb8, b), c, 0, 0, 0);
    }
    static __device__ inline xf4 mma16(xu4 a, xu4 b, xf4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(xb8, a), __builtin_bit_cast(xb8, b), c, 0, 0, 0);
    }
    static __device__ inline S put(float v) { return (__bf16)v; }
};

// 16 bytes shifted by one value
template <typename X>
__device__ inline xu4 exp_down(xu4 r) {
    if constexpr (X::kVec == 4) return xu4{r[1], r[2], r[3], 0u};
    return xu4{r[0] >> 16 | r[1] << 16, r[1] >> 16 | r[2] << 16, r[2] >> 16 | r[3] << 16, r[3] >> 16};
}
template <typename X>
__device__ inline xu4 exp_up(xu4 r) {
    if constexpr (X::kVec == 4) return xu4{0u, r[0], r[1], r[2]};
    return xu4{r[0] << 16, r[0] >> 16 | r[1] << 16, r[1] >> 16 | r[2] << 16, r[2] >> 16 | r[3] << 16};
}
// kVec values at p, of which `left` (any number, below 1: none) are inside; zeros past them.  Fewer than all go one by
// one through loops, which keep the code and its masks small.
template <typename X>
__device__ inline xu4 exp_load(const uint8_t* p, int left) {
    if (left >= X::kVec) return *reinterpret_cast<const xu4u*>(p);
    xu4 r = {0u, 0u, 0u, 0u};
#pragma nounroll
    for (int j = left - 1; j >= 0; --j) {
        r = exp_up<X>(r);
        if constexpr (X::kVec == 4) r[0] = reinterpret_cast<const uint32_t*>(p)[j];
        else r[0] |= reinterpret_cast<const uint16_t*>(p)[j];
    }
    return r;
}
template <typename X>
__device__ inline void exp_store(uint8_t* p, xu4 r, int left) {
    if (left >= X::kVec) {
        *reinterpret_cast<xu4u*>(p) = r;
        return;
    }
#pragma nounroll
    for (int j = 0; j < left; ++j) {
        if constexpr (X::kVec == 4) reinterpret_cast<uint32_t*>(p)[j] = r[0];
        else reinterpret_cast<uint16_t*>(p)[j] = (uint16_t)r[0];
        r = exp_down<X>(r);
    }
}

// ---------------------------------------------------------------------------
// groups
// ---------------------------------------------------------------------------
// What a caller's groups buffer holds, in 32-bit words.  The head says which call it was made for: a kernel given
// groups of another shape, or never made, sets the sticky error word and ends.
constexpr int kExpHead = 16;
constexpr uint32_t kExpMagic = 0x67727031u;
constexpr int kExpSmall = 16, kExpTile = 128;     // rows of the two lists' tiles
constexpr int kExpChunk = 4096;                   // rows that a workgroup of k_expert_count / _place sorts
constexpr int kExpMaxExperts = 4096;
constexpr unsigned kErrExpertId = 1u, kErrExpertGroups = 5u;
struct ExpertPlan {
    int n_rows, n_ids, n_experts, chunks;
    size_t off, order, small, tiles, counts, words;   // in words from the buffer's start
    int max_small, max_tiles;
};
inline ExpertPlan expert_plan(int n_ids, int n_tokens, int n_experts) {
    ExpertPlan p{};
    p.n_rows = n_ids * n_tokens;
    p.n_ids = n_ids;
    p.n_experts = n_experts;
    p.chunks = (p.n_rows + kExpChunk - 1) / kExpChunk;
    const int groups = p.n_rows < n_experts + 2 ? p.n_rows : n_experts + 2;
    p.max_small = p.n_rows / kExpSmall + groups;
    p.max_tiles = p.n_rows / kExpTile + groups;
    auto take = [&](size_t n) {
        const size_t at = p.words;
        p.words += (n + 3) / 4 * 4;
        return at;
    };
    p.words = kExpHead;
    p.off = take(n_experts + 3);                      // positions where each expert's rows begin; then rows of -1, of bad ids
    p.order = take(p.n_rows);                         // the rows in that order
    p.small = take((size_t)p.max_small * 4);          // tiles (expert, first position, rows, 0); expert -1, -2: none, bad
    p.tiles = take((size_t)p.max_tiles * 4);
    p.counts = take(p.chunks > 1 ? (size_t)p.chunks * (n_experts + 2) : 0);
    return p;
}
// words of the head
constexpr int kExpHeadMagic = 0, kExpHeadRows = 1, kExpHeadIds = 2, kExpHeadExperts = 3, kExpHeadSmall = 4, kExpHeadTiles = 5;

struct ExpertGroupArgs {
    const uint8_t* ids;
    size_t ids_id, ids_tok;
    uint32_t* g;
    ExpertPlan p;
    unsigned int* err;
};

__device__ inline int exp_key(const ExpertGroupArgs& a, int row) {
    const int t = row / a.p.n_ids, i = row - t * a.p.n_ids;
    const int e = *reinterpret_cast<const int*>(a.ids + (size_t)t * a.ids_tok + (size_t)i * a.ids_id);
    return e >= 0 && e < a.p.n_experts ? e : e == -1 ? a.p.n_experts : a.p.n_experts + 1;
}

constexpr int kExpGroupThreads = 1024, kExpGroupWaves = kExpGroupThreads / 64;
constexpr int kExpWaveRows = kExpChunk / kExpGroupWaves, kExpWaveSteps = kExpWaveRows / 64;

// A chunk's rows, each wave its own run of them: counts of each wave and key in LDS (16 bits, two to a word)
__device__ inline void exp_read_keys(const ExpertGroupArgs& a, int chunk, int (&key)[kExpWaveSteps]) {
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int first = chunk * kExpChunk + wave * kExpWaveRows;
#pragma unroll
    for (int s = 0; s < kExpWaveSteps; ++s) {
        const int row = first + s * 64 + lane;
        key[s] = row < a.p.n_rows ? exp_key(a, row) : -1;
    }
}

__device__ inline int exp_block_scan(int v, int* tmp, int& total) {    // exclusive, over kExpGroupThreads
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    int s = v;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int o = __shfl_up(s, d);
        if (lane >= d) s += o;
    }
    __syncthreads();
    if (lane == 63) tmp[wave] = s;
    __syncthreads();
    int before = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < kExpGroupWaves; ++w) {
        if (w < wave) before += tmp[w];
        total += tmp[w];
    }
    return before + s - v;
}

__global__ __launch_bounds__(kExpGroupThreads) void k_expert_count(ExpertGroupArgs a) {
    extern __shared__ int exp_lds[];
    const int keys = a.p.n_experts + 2;
    for (int e = threadIdx.x; e < keys; e += kExpGroupThreads) exp_lds[e] = 0;
    int key[kExpWaveSteps];
    exp_read_keys(a, blockIdx.x, key);
    __syncthreads();
#pragma unroll
    for (int s = 0; s < kExpWaveSteps; ++s)
        if (key[s] >= 0) atomicAdd(&exp_lds[key[s]], 1);
    __syncthreads();
    for (int e = threadIdx.x; e < keys; e += kExpGroupThreads) a.g[a.p.counts + (size_t)blockIdx.x * keys + e] = exp_lds[e];
}

// The keys' first positions and their tiles, from cnt(e), by one workgroup.  base(e, at): where key e begins
template <typename Count, typename Base>
__device__ inline void exp_lists(const ExpertGroupArgs& a, int* tmp, Count cnt, Base base) {
    const int E = a.p.n_experts, keys = E + 2;
    const int seg = (keys + kExpGroupThreads - 1) / kExpGroupThreads;
    const int e0 = min(keys, (int)threadIdx.x * seg), e1 = min(keys, e0 + seg);
    int rows = 0, small = 0, tiles = 0, total;
    for (int e = e0; e < e1; ++e) {
        const int c = cnt(e);
        rows += c;
        small += (c + kExpSmall - 1) / kExpSmall;
        tiles += (c + kExpTile - 1) / kExpTile;
    }
    int at = exp_block_scan(rows, tmp, total);
    int s = exp_block_scan(small, tmp, total);
    const int n_small = total;
    int t = exp_block_scan(tiles, tmp, total);
    int4* ls = reinterpret_cast<int4*>(a.g + a.p.small);
    int4* lt = reinterpret_cast<int4*>(a.g + a.p.tiles);
    for (int e = e0; e < e1; ++e) {
        const int c = cnt(e), who = e < E ? e : E - 1 - e;
        a.g[a.p.off + e] = at;
        for (int o = 0; o < c; o += kExpSmall) ls[s++] = make_int4(who, at + o, min(kExpSmall, c - o), 0);
        for (int o = 0; o < c; o += kExpTile) lt[t++] = make_int4(who, at + o, min(kExpTile, c - o), 0);
        base(e, at);
        at += c;
        if (e == E + 1 && c) *reinterpret_cast<volatile unsigned int*>(a.err) = kErrExpertId;
    }
    if (threadIdx.x == 0) {
        a.g[a.p.off + keys] = a.p.n_rows;
        a.g[kExpHeadMagic] = kExpMagic;
        a.g[kExpHeadRows] = a.p.n_rows;
        a.g[kExpHeadIds] = a.p.n_ids;
        a.g[kExpHeadExperts] = E;
        a.g[kExpHeadSmall] = n_small;
        a.g[kExpHeadTiles] = total;
    }
}

// Several chunks: the counts of each become where its rows of a key begin
__global__ __launch_bounds__(kExpGroupThreads) void k_expert_scan(ExpertGroupArgs a) {
    __shared__ int tmp[kExpGroupWaves];
    extern __shared__ int exp_lds[];
    const int keys = a.p.n_experts + 2;
    uint32_t* counts = a.g + a.p.counts;
    for (int e = threadIdx.x; e < keys; e += kExpGroupThreads) {
        int s = 0;
        for (int c = 0; c < a.p.chunks; ++c) s += (int)counts[(size_t)c * keys + e];
        exp_lds[e] = s;
    }
    __syncthreads();
    exp_lists(a, tmp, [&](int e) { return exp_lds[e]; }, [&](int e, int at) {
        for (int c = 0; c < a.p.chunks; ++c) {
            const int n = (int)counts[(size_t)c * keys + e];
            counts[(size_t)c * keys + e] = (uint32_t)at;
            at += n;
        }
    });
}

// The rows' places.  ALONE: the one chunk of a small call, whose lists are made here too.
template <bool ALONE>
__global__ __launch_bounds__(kExpGroupThreads) void k_expert_place(ExpertGroupArgs a) {
    extern __shared__ int exp_lds[];                  // [waves][words] counts of 16 bits; [keys] starts; scan
    const int keys = a.p.n_experts + 2, words = (keys + 1) / 2;
    uint32_t* hist = reinterpret_cast<uint32_t*>(exp_lds);
    int* start = exp_lds + kExpGroupWaves * words;
    int* tmp = start + keys;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    for (int e = threadIdx.x; e < kExpGroupWaves * words; e += kExpGroupThreads) hist[e] = 0;
    int key[kExpWaveSteps];
    exp_read_keys(a, blockIdx.x, key);
    __syncthreads();
    uint32_t* mine = hist + wave * words;
#pragma unroll
    for (int s = 0; s < kExpWaveSteps; ++s)
        if (key[s] >= 0) atomicAdd(&mine[key[s] >> 1], 1u << (16 * (key[s] & 1)));
    __syncthreads();
    // counts -> how many of the key the waves before have; a word's two keys at once (no carry: 4,096 rows at most)
    for (int w = threadIdx.x; w < words; w += kExpGroupThreads) {
        uint32_t sum = 0;
#pragma unroll
        for (int v = 0; v < kExpGroupWaves; ++v) {
            const uint32_t c = hist[v * words + w];
            hist[v * words + w] = sum;
            sum += c;
        }
        if constexpr (ALONE) {
            start[2 * w] = (int)(sum & 0xFFFFu);
            if (2 * w + 1 < keys) start[2 * w + 1] = (int)(sum >> 16);
        }
    }
    __syncthreads();
    if constexpr (ALONE) {
        exp_lists(a, tmp, [&](int e) { return start[e]; }, [&](int e, int at) { start[e] = at; });
    } else {
        for (int e = threadIdx.x; e < keys; e += kExpGroupThreads) start[e] = (int)a.g[a.p.counts + (size_t)blockIdx.x * keys + e];
    }
    __syncthreads();
    const int first = blockIdx.x * kExpChunk + wave * kExpWaveRows;
    uint16_t* taken = reinterpret_cast<uint16_t*>(mine);
    const int bits = 32 - __builtin_clz(keys);
#pragma unroll
    for (int s = 0; s < kExpWaveSteps; ++s) {
        const bool some = key[s] >= 0;
        uint64_t same = __ballot(some);               // lanes with this lane's key
        for (int b = 0; b < bits; ++b) {
            const uint64_t set = __ballot((key[s] >> b) & 1);
            same &= (key[s] >> b) & 1 ? set : ~set;
        }
        if (some) {
            const int before = __builtin_popcountll(same & ((1ull << lane) - 1));
            const int n = taken[key[s]];
            a.g[a.p.order + start[key[s]] + n + before] = (uint32_t)(first + s * 64 + lane);
            __builtin_amdgcn_wave_barrier();
            if (before == 0) taken[key[s]] = (uint16_t)(n + __builtin_popcountll(same));
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");   // the next step's lanes read what this one's left
        __builtin_amdgcn_wave_barrier();
    }
}

// ---------------------------------------------------------------------------
// products
// ---------------------------------------------------------------------------
struct ExpertArgs {
    const uint32_t* g;
    ExpertPlan p;
    const uint8_t* w;                 // [n_experts][rows][k]
    int k, rows;
    const uint8_t* x;                 // row (t, i): x + t * x_tok + (i % x_rows) * x_id
    size_t x_id, x_tok;
    int x_rows;
    const uint8_t* dy;                // row (t, i): dy + t * dy_tok + i * dy_id
    size_t dy_id, dy_tok;
    uint8_t* out;                     // y or dx
    size_t out_id, out_tok;
    float* dw;                        // [n_experts][rows][k]
    int add;
    unsigned int* err;
};

__device__ inline bool exp_groups_fit(const ExpertArgs& a) {
    const bool ok = a.g[kExpHeadMagic] == kExpMagic && a.g[kExpHeadRows] == (uint32_t)a.p.n_rows &&
                    a.g[kExpHeadIds] == (uint32_t)a.p.n_ids && a.g[kExpHeadExperts] == (uint32_t)a.p.n_experts;
    if (!ok && threadIdx.x == 0) *reinterpret_cast<volatile unsigned int*>(a.err) = kErrExpertGroups;
    return ok;
}
__device__ inline const uint8_t* exp_row_x(const ExpertArgs& a, uint32_t row) {
    const uint32_t t = row / (uint32_t)a.p.n_ids, i = row - t * (uint32_t)a.p.n_ids;
    return a.x + (size_t)t * a.x_tok + (a.x_rows == 1 ? 0 : (size_t)i * a.x_id);
}
__device__ inline const uint8_t* exp_row_dy(const ExpertArgs& a, uint32_t row) {
    const uint32_t t = row / (uint32_t)a.p.n_ids, i = row - t * (uint32_t)a.p.n_ids;
    return a.dy + (size_t)t * a.dy_tok + (size_t)i * a.dy_id;
}
__device__ inline uint8_t* exp_row_out(const ExpertArgs& a, uint32_t row) {
    const uint32_t t = row / (uint32_t)a.p.n_ids, i = row - t * (uint32_t)a.p.n_ids;
    return a.out + (size_t)t * a.out_tok + (size_t)i * a.out_id;
}
// Workgroups are dealt to the 8 dies in turn; each die takes a run of the work, so that an expert's tiles, which read
// the same weights, and a tile's columns, which read the same rows, meet in one die's L2.  False: nothing left.
__device__ inline bool exp_work(int id, int all, int& work) {
    const int each = (all + 7) / 8, q = id >> 3;
    work = (id & 7) * each + q;
    return q < each && work < all;
}
// rows without an expert (zeros), or with a bad id (NaN)
template <typename X>
__device__ inline void exp_fill(const ExpertArgs& a, const int4& it, int col0, int cols, int width) {
    const float v = it.x == -1 ? 0.0f : __builtin_nanf("");
    const int n = min(cols, width - col0);
    for (int m = 0; m < it.z; ++m) {
        typename X::S* o = reinterpret_cast<typename X::S*>(exp_row_out(a, a.g[a.p.order + it.y + m])) + col0;
        for (int c = threadIdx.x; c < n; c += blockDim.x) o[c] = X::put(v);
    }
}

constexpr int kExpThreads = 256;
constexpr int kModeForward = 0, kModeDx = 1, kModeDw = 2;

// A tile of BM x BN outputs, four waves of (BM / 2) x (BN / 2), the summed axis in steps of 128 bytes.
//   forward: rows of x by rows of W;  dx: rows of dy by columns of W;  dw: columns of dy by columns of x, summed over a
//   group's rows.
// An operand whose summed axis is contiguous in memory lies in LDS as rows of 128 bytes, its 16-byte chunks
// permuted by the row's low bits (any 8 neighbouring lanes of a read then cover all banks); one whose summed axis is
// strided lies as BK rows of the tile's columns, and its fragments are transposed as they are read
// (ds_read_b64_tr_b16: 16 lanes read a 4 x 16 block and get its columns); f32 values are read one by one.
template <typename X, int MODE>
struct ExpGemm {
    typedef typename X::S S;
    static constexpr int BM = kExpTile, BN = 128, BK = 128 / (int)sizeof(S), VEC = X::kVec, ES = (int)sizeof(S);
    static constexpr bool TA = MODE == kModeDw, TB = MODE != kModeForward;
    static constexpr int kSide = 128 * 128;           // bytes of one operand's tile
    static constexpr int kLds = 4 * kSide;            // two operands, two buffers
    static constexpr int kOutStride = BN * ES + 16;
    static constexpr int kLdsAll = MODE == kModeDw || kLds >= BM * kOutStride ? kLds : BM * kOutStride;
    static constexpr int CPR = 128 * ES / 16;         // 16-byte chunks of a strided operand's row

    static __device__ inline int at_contiguous(int row, int chunk) { return row * 128 + ((chunk ^ (row & 7)) << 4); }
    static __device__ inline int at_strided(int row, int chunk) {
        return row * (128 * ES) + ((ES == 2 ? chunk ^ ((row & 3) << 1) : chunk) << 4);
    }
    // the fragment of 32 rows (or columns) from r0, step s of the tile's
    static __device__ inline xu4 contiguous(const uint8_t* t, int r0, int s) {
        const int lane = threadIdx.x & 63;
        return *reinterpret_cast<const xu4*>(t + at_contiguous(r0 + (lane & 31), 2 * s + (lane >> 5)));
    }
    static __device__ inline xu4 strided(const uint8_t* t, int c0, int s) {
        const int lane = threadIdx.x & 63;
        xu4 r;
        if constexpr (ES == 2) {
            const int l = lane & 15, row = s * 16 + (lane >> 5) * 8 + (l >> 2), col = c0 + (lane & 16) + (l & 3) * 4;
            const uint8_t* p = t + at_strided(row, col >> 3) + ((col & 4) << 1);
            typedef __attribute__((address_space(3))) xs4 lds_xs4;
            const xs4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_xs4*)(p));
            const xs4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_xs4*)(p + 4 * 128 * ES));
            __builtin_memcpy(&r, &lo, 8);
            __builtin_memcpy(reinterpret_cast<char*>(&r) + 8, &hi, 8);
        } else {
            xf4 v;
#pragma unroll
            for (int j = 0; j < 4; ++j)
                v[j] = *reinterpret_cast<const float*>(t + (s * 8 + (lane >> 5) * 4 + j) * (128 * ES) + (c0 + (lane & 31)) * ES);
            r = __builtin_bit_cast(xu4, v);
        }
        return r;
    }
};

template <typename X, int MODE>
__global__ __launch_bounds__(kExpThreads, 2) void k_expert_gemm(ExpertArgs a) {
    typedef ExpGemm<X, MODE> G;
    constexpr int ES = G::ES, VEC = G::VEC, BK = G::BK, BM = G::BM, BN = G::BN;
    extern __shared__ __align__(16) uint8_t exp_tile[];
    if (!exp_groups_fit(a)) return;
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    // the tile: an expert's rows (or the rows that a sum goes over), output rows from m0 and columns from n0
    const int width = MODE == kModeForward ? a.rows : a.k;             // of an output row
    const int col_tiles = (width + BN - 1) / BN;
    int work, expert, first, count, m0 = 0, n0;
    if constexpr (MODE == kModeDw) {
        const int row_tiles = (a.rows + BM - 1) / BM;
        if (!exp_work(blockIdx.x, a.p.n_experts * row_tiles * col_tiles, work)) return;
        expert = work / (row_tiles * col_tiles);
        work -= expert * row_tiles * col_tiles;
        m0 = work / col_tiles * BM;
        n0 = work % col_tiles * BN;
        first = (int)a.g[a.p.off + expert];
        count = (int)a.g[a.p.off + expert + 1] - first;
        if (count == 0 && a.add) return;
    } else {
        if (!exp_work(blockIdx.x, (int)a.g[kExpHeadTiles] * col_tiles, work)) return;
        const int4 it = reinterpret_cast<const int4*>(a.g + a.p.tiles)[work / col_tiles];
        n0 = work % col_tiles * BN;
        if (it.x < 0) {
            exp_fill<X>(a, it, n0, BN, width);
            return;
        }
        expert = it.x;
        first = it.y;
        count = it.z;
    }
    const uint32_t* order = a.g + a.p.order + first;
    const uint8_t* w = a.w + (size_t)expert * a.rows * a.k * ES;
    const int K = MODE == kModeForward ? a.k : MODE == kModeDx ? a.rows : count;   // length of the sum

    // what this thread stages: of a contiguous operand chunk c of rows r, r + 32, ..; of a strided one chunk c of
    // every (256 / CPR)th row
    constexpr int NL = 4;                             // 16-byte loads of an operand's tile for a thread
    constexpr int RPI = kExpThreads / G::CPR;         // rows between two of them
    const uint8_t *pa[NL], *pb[NL];
    const int cc = tid & 7, rc = tid >> 3, cs = tid % G::CPR, rs = tid / G::CPR;
    if constexpr (MODE != kModeDw) {
#pragma unroll
        for (int i = 0; i < NL; ++i) {                // rows past the tile repeat its first and are not stored
            const int m = rc + 32 * i;
            const uint32_t row = order[m < count ? m : 0];
            pa[i] = (MODE == kModeForward ? exp_row_x(a, row) : exp_row_dy(a, row)) + cc * 16;
        }
    }
    if constexpr (MODE == kModeForward) {
#pragma unroll
        for (int i = 0; i < NL; ++i) pb[i] = w + (size_t)min(n0 + rc + 32 * i, a.rows - 1) * a.k * ES + cc * 16;
    }
    xu4 ra[NL], rb[NL];
    auto load = [&](int k0) {
#pragma unroll
        for (int i = 0; i < NL; ++i) {
            if constexpr (MODE != kModeDw) ra[i] = exp_load<X>(pa[i] + (size_t)k0 * ES, K - k0 - cc * VEC);
            if constexpr (MODE == kModeForward) rb[i] = exp_load<X>(pb[i] + (size_t)k0 * ES, K - k0 - cc * VEC);
            if constexpr (MODE == kModeDx) {
                const int n = k0 + rs + RPI * i, col = n0 + cs * VEC;
                rb[i] = exp_load<X>(w + ((size_t)n * a.k + col) * ES, n < K ? a.k - col : 0);
            }
            if constexpr (MODE == kModeDw) {
                const int r = k0 + rs + RPI * i, ca = m0 + cs * VEC, cb = n0 + cs * VEC;
                const uint32_t row = order[r < K ? r : 0];
                ra[i] = exp_load<X>(exp_row_dy(a, row) + (size_t)ca * ES, r < K ? a.rows - ca : 0);
                rb[i] = exp_load<X>(exp_row_x(a, row) + (size_t)cb * ES, r < K ? a.k - cb : 0);
            }
        }
    };
    auto stage = [&](int buf) {
        uint8_t* ta = exp_tile + buf * 2 * G::kSide;
        uint8_t* tb = ta + G::kSide;
#pragma unroll
        for (int i = 0; i < NL; ++i) {
            *reinterpret_cast<xu4*>(ta + (G::TA ? G::at_strided(rs + RPI * i, cs) : G::at_contiguous(rc + 32 * i, cc))) = ra[i];
            *reinterpret_cast<xu4*>(tb + (G::TB ? G::at_strided(rs + RPI * i, cs) : G::at_contiguous(rc + 32 * i, cc))) = rb[i];
        }
    };
    const int wm = (wave >> 1) * 64, wn = (wave & 1) * 64;
    xf16 acc[2][2] = {};
    const int steps = (K + BK - 1) / BK;
    if (steps) {
        load(0);
        stage(0);
        __syncthreads();
    }
    for (int t = 0; t < steps; ++t) {
        if (t + 1 < steps) load((t + 1) * BK);
        const uint8_t* ta = exp_tile + (t & 1) * 2 * G::kSide;
        const uint8_t* tb = ta + G::kSide;
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            xu4 fa[2], fb[2];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                fa[j] = G::TA ? G::strided(ta, wm + 32 * j, s) : G::contiguous(ta, wm + 32 * j, s);
                fb[j] = G::TB ? G::strided(tb, wn + 32 * j, s) : G::contiguous(tb, wn + 32 * j, s);
            }
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j) acc[i][j] = X::mma32(fa[i], fb[j], acc[i][j]);
        }
        if (t + 1 < steps) stage((t + 1) & 1);
        __syncthreads();
    }
    // of a 32 x 32 result a lane has column lane % 32 and rows 8 (v / 4) + 4 (lane / 32) + v % 4
    if constexpr (MODE == kModeDw) {
        float* dw = a.dw + (size_t)expert * a.rows * a.k;
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int n = n0 + wn + 32 * j + (lane & 31);
#pragma unroll
                for (int v = 0; v < 16; ++v) {
                    const int m = m0 + wm + 32 * i + 8 * (v >> 2) + 4 * (lane >> 5) + (v & 3);
                    if (m < a.rows && n < a.k) {
                        float* o = dw + (size_t)m * a.k + n;
                        *o = a.add ? *o + acc[i][j][v] : acc[i][j][v];
                    }
                }
            }
    } else {
        // through LDS, so that a row's columns are stored 16 bytes a lane
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int v = 0; v < 16; ++v) {
                    const int m = wm + 32 * i + 8 * (v >> 2) + 4 * (lane >> 5) + (v & 3), n = wn + 32 * j + (lane & 31);
                    *reinterpret_cast<typename X::S*>(exp_tile + m * G::kOutStride + n * ES) = X::put(acc[i][j][v]);
                }
        __syncthreads();
        constexpr int CPO = BN * ES / 16;
        for (int c = tid; c < count * CPO; c += kExpThreads) {
            const int m = c / CPO, n = c % CPO * VEC;
            exp_store<X>(exp_row_out(a, order[m]) + (size_t)(n0 + n) * ES,
                         *reinterpret_cast<const xu4*>(exp_tile + m * G::kOutStride + n * ES), width - n0 - n);
        }
    }
}

// Few rows: a workgroup has up to 16 rows of one expert and NT * 16 rows of its W; its waves share k.  W's rows go
// from memory into MFMA operands (a lane has 16 bytes of row lane % 16), x's rows likewise from L2; the waves' sums meet
// in LDS, added in the waves' order.
constexpr int kExpRowsWaves = 8;
template <typename X, int NT>
__global__ __launch_bounds__(64 * kExpRowsWaves) void k_expert_rows(ExpertArgs a) {
    constexpr int ES = (int)sizeof(typename X::S), VEC = X::kVec, COLS = 16 * NT, STEP = 4 * VEC, U = 4;
    __shared__ xf4 part[kExpRowsWaves][NT][64];
    if (!exp_groups_fit(a)) return;
    const int col_tiles = (a.rows + COLS - 1) / COLS;
    int work;
    if (!exp_work(blockIdx.x, (int)a.g[kExpHeadSmall] * col_tiles, work)) return;
    const int4 it = reinterpret_cast<const int4*>(a.g + a.p.small)[work / col_tiles];
    const int n0 = work % col_tiles * COLS;
    if (it.x < 0) {
        exp_fill<X>(a, it, n0, COLS, a.rows);
        return;
    }
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, r = lane & 15, q = lane >> 4;
    const uint32_t row = a.g[a.p.order + it.y + min(r, it.z - 1)];
    const uint8_t* px = exp_row_x(a, row) + q * 16;
    const uint8_t* pw[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t)
        pw[t] = a.w + ((size_t)it.x * a.rows + min(n0 + 16 * t + r, a.rows - 1)) * a.k * ES + q * 16;
    // each wave a run of steps
    const int steps = (a.k + STEP - 1) / STEP, each = (steps + kExpRowsWaves - 1) / kExpRowsWaves;
    const int s0 = min(steps, wave * each), s1 = min(steps, s0 + each);
    xf4 acc[NT] = {};
    int s = s0;
    for (; s + U <= s1 && (s + U) * STEP <= a.k; s += U) {
        xu4 fx[U], fw[NT][U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
#pragma unroll
            for (int t = 0; t < NT; ++t) fw[t][u] = *reinterpret_cast<const xu4u*>(pw[t] + (size_t)(s + u) * 64);
            fx[u] = *reinterpret_cast<const xu4u*>(px + (size_t)(s + u) * 64);
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int t = 0; t < NT; ++t) acc[t] = X::mma16(fw[t][u], fx[u], acc[t]);
    }
    for (; s < s1; ++s) {
        const int left = a.k - s * STEP - q * VEC;
        const xu4 fx = exp_load<X>(px + (size_t)s * 64, left);
#pragma unroll
        for (int t = 0; t < NT; ++t) acc[t] = X::mma16(exp_load<X>(pw[t] + (size_t)s * 64, left), fx, acc[t]);
    }
#pragma unroll
    for (int t = 0; t < NT; ++t) part[wave][t][lane] = acc[t];
    __syncthreads();
    // a lane has four neighbouring columns of one row
    for (int c = threadIdx.x; c < NT * 64; c += 64 * kExpRowsWaves) {
        const int t = c >> 6, l = c & 63;
        xf4 v = part[0][t][l];
#pragma unroll
        for (int w = 1; w < kExpRowsWaves; ++w) v += part[w][t][l];
        const int m = l & 15, n = n0 + 16 * t + 4 * (l >> 4);
        if (m >= it.z) continue;
        typename X::S* o = reinterpret_cast<typename X::S*>(exp_row_out(a, a.g[a.p.order + it.y + m])) + n;
        typename X::S s4[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) s4[j] = X::put(v[j]);
        if (n + 4 <= a.rows) {
            if constexpr (ES == 4) {
                *reinterpret_cast<xu4u*>(o) = __builtin_bit_cast(xu4, s4);
            } else {
                *reinterpret_cast<xu2u*>(o) = __builtin_bit_cast(xu2, s4);
            }
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (n + j < a.rows) o[j] = s4[j];
        }
    }
}

}  // namespace sabah
