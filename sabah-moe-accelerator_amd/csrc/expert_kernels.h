// Products of experts kept in float types (f32, f16, bf16), grouped by expert with ragged sizes, and
// their gradients.  Row r = t * n_ids + i is (token t, slot i); e_r = ids[t][i], -1: none.
//   forward    y_r = W[e_r] x_r
//   backward   dx_r = W[e_r]^T dy_r;   dW[e] (+)= sum over the rows of e of dy_r x_r^T
// Products of 16-bit values are exact where f32 has them (24 bits, from 2^-149), f32's are rounded; subnormal operands count as what
// they are; sums are f32 on the matrix cores; y and dx are rounded once, dW is f32.
//
// k_expert_group_few, _count, _scan, _place: the rows in expert order, stable and without an order that depends on
//   atomics, so the same ids give the same bits; cut into tiles of one expert.
// k_expert_rows:  up to 16 rows of one expert (decode, few tokens): W streamed from HBM into MFMA operands.  HBM bounds it:
//   47 tokens of 8 of 128 experts (385 MB) in 79 us, the rate of a large copy.
// k_expert_fast, k_expert_dw: tiles whose operands go from memory straight into LDS.  Bounds, at 2,048 -> 768 in bf16:
//   over 8 experts of 8,192 rows 211 us (976 TFLOP/s; the same products with nothing to load 148, the loads alone 139:
//   what is left is the two getting in each other's way); over 128 experts of 512 rows the weights' 402 MB come at half the
//   rate of a copy, because two tiles ask for the same bytes at once, which leaves half as many different ones under way.
//   dW of 128 experts writes 805 MB: 338 us, where the sums alone take 214 - 239 and the loads alone 140.
// k_expert_gemm:  the same products for rows at any alignment, staged through registers.
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
// The same from column c of a row of `width` >= kVec, without a branch for each value: a chunk that the row ends in, or one past
// it, is read as the row's last kVec values (exp_last) and shifted down by what lies past the end (exp_over bytes).
template <typename X>
__device__ inline xu4 exp_last(const uint8_t* row, int c, int width) {
    return *reinterpret_cast<const xu4u*>(row + (size_t)min(c, width - X::kVec) * sizeof(typename X::S));
}
template <typename X>
__device__ inline int exp_over(int c, int width) {
    return max(0, min(c + X::kVec - width, X::kVec)) * (int)sizeof(typename X::S);
}
__device__ inline xu4 exp_shift(xu4 r, int over) {
    if (over) {
        if (over & 8) r = xu4{r[2], r[3], 0u, 0u};
        if (over & 4) r = xu4{r[1], r[2], r[3], 0u};
        if (over & 2) r = xu4{r[0] >> 16 | r[1] << 16, r[1] >> 16 | r[2] << 16, r[2] >> 16 | r[3] << 16, r[3] >> 16};
        if (over & 16) r = xu4{0u, 0u, 0u, 0u};
    }
    return r;
}
template <typename X>
__device__ inline xu4 exp_chunk(const uint8_t* row, int c, int width) {
    return exp_shift(exp_last<X>(row, c, width), exp_over<X>(c, width));
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
constexpr int kExpSmall = 16, kExpTile = 128, kExpLarge = 256;   // rows of the three lists' tiles
constexpr int kExpChunk = 4096;                   // rows that a workgroup of k_expert_count / _place sorts
constexpr int kExpMaxExperts = 4096;
// Rows to an expert, on average, up to which a forward call streams its weights (k_expert_rows) and has small tiles.  us of
// the two at 2,048 -> 768 of 128 experts in bf16: 72.6 and 86.1 at 2 rows, 95.7 and 101 at 8, 117 and 105 at 16.  By the average,
// which the host knows: 1,280 rows that all have one of the 128 take 35 us as 80 small tiles, 29 as large ones
constexpr int kExpFewRows = 10;
constexpr unsigned kErrExpertId = 1u, kErrExpertGroups = 5u;
struct ExpertPlan {
    int n_rows, n_ids, n_experts, chunks;
    size_t off, order, small, tiles, large, counts, words;   // in words from the buffer's start
    int max_small, max_tiles, max_large;
};
inline ExpertPlan expert_plan(int n_ids, int n_tokens, int n_experts) {
    ExpertPlan p{};
    p.n_rows = n_ids * n_tokens;
    p.n_ids = n_ids;
    p.n_experts = n_experts;
    p.chunks = (p.n_rows + kExpChunk - 1) / kExpChunk;
    const int groups = p.n_rows < n_experts + 2 ? p.n_rows : n_experts + 2;
    p.max_small = p.n_rows <= (long long)kExpFewRows * n_experts ? p.n_rows / kExpSmall + groups : 0;
    p.max_tiles = p.n_rows / kExpTile + groups;
    p.max_large = p.n_rows / kExpLarge + groups;
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
    p.large = take((size_t)p.max_large * 4);
    p.counts = take(p.chunks > 1 ? (size_t)p.chunks * (n_experts + 2) : 0);
    return p;
}
// words of the head
constexpr int kExpHeadMagic = 0, kExpHeadRows = 1, kExpHeadIds = 2, kExpHeadExperts = 3, kExpHeadSmall = 4, kExpHeadTiles = 5, kExpHeadLarge = 6;

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

__device__ inline uint64_t exp_block_scan(uint64_t v, uint64_t* tmp, uint64_t& total) {    // exclusive, over kExpGroupThreads
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    uint64_t s = v;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const uint64_t o = __shfl_up((unsigned long long)s, d);
        if (lane >= d) s += o;
    }
    __syncthreads();
    if (lane == 63) tmp[wave] = s;
    __syncthreads();
    uint64_t before = 0;
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

__device__ inline void exp_head(const ExpertGroupArgs& a, int small, int tiles, int large) {
    a.g[a.p.off + a.p.n_experts + 2] = a.p.n_rows;
    a.g[kExpHeadMagic] = kExpMagic;
    a.g[kExpHeadRows] = a.p.n_rows;
    a.g[kExpHeadIds] = a.p.n_ids;
    a.g[kExpHeadExperts] = a.p.n_experts;
    a.g[kExpHeadSmall] = small;
    a.g[kExpHeadTiles] = tiles;
    a.g[kExpHeadLarge] = large;
}
constexpr int exp_tiles(int rows, int of) { return (rows + of - 1) / of; }

// The keys' first positions and, where WRITE, their tiles, from cnt(e), by one workgroup.  base(e, at): where key e begins
template <typename Count, typename Base>
__device__ inline void exp_lists(const ExpertGroupArgs& a, uint64_t* tmp, bool write, Count cnt, Base base) {
    const int E = a.p.n_experts, keys = E + 2;
    const int seg = (keys + kExpGroupThreads - 1) / kExpGroupThreads;
    const int e0 = min(keys, (int)threadIdx.x * seg), e1 = min(keys, e0 + seg);
    uint64_t one = 0, two = 0, total, total2 = 0;               // rows and small tiles, tiles and large ones: 32 bits each
    for (int e = e0; e < e1; ++e) {
        const int c = cnt(e);
        one += (uint64_t)c | (a.p.max_small ? (uint64_t)exp_tiles(c, kExpSmall) << 32 : 0);
        two += (uint64_t)exp_tiles(c, kExpTile) | (uint64_t)exp_tiles(c, kExpLarge) << 32;
    }
    one = exp_block_scan(one, tmp, total);
    if (write) two = exp_block_scan(two, tmp, total2);          // uniform
    int at = (int)(uint32_t)one, s = (int)(one >> 32), t = (int)(uint32_t)two, l = (int)(two >> 32);
    int4* ls = reinterpret_cast<int4*>(a.g + a.p.small);
    int4* lt = reinterpret_cast<int4*>(a.g + a.p.tiles);
    int4* ll = reinterpret_cast<int4*>(a.g + a.p.large);
    for (int e = e0; e < e1; ++e) {
        const int c = cnt(e), who = e < E ? e : E - 1 - e;
        if (write) {
            a.g[a.p.off + e] = at;
            if (a.p.max_small)
                for (int o = 0; o < c; o += kExpSmall) ls[s++] = make_int4(who, at + o, min(kExpSmall, c - o), 0);
            for (int o = 0; o < c; o += kExpTile) lt[t++] = make_int4(who, at + o, min(kExpTile, c - o), 0);
            for (int o = 0; o < c; o += kExpLarge) ll[l++] = make_int4(who, at + o, min(kExpLarge, c - o), 0);
            if (e == E + 1 && c) *reinterpret_cast<volatile unsigned int*>(a.err) = kErrExpertId;
        }
        base(e, at);
        at += c;
    }
    if (write && threadIdx.x == 0) exp_head(a, (int)(total >> 32), (int)(uint32_t)total2, (int)(total2 >> 32));
}

// Many chunks: the counts of each become where its rows of a key begin
__global__ __launch_bounds__(kExpGroupThreads) void k_expert_scan(ExpertGroupArgs a) {
    __shared__ uint64_t tmp[kExpGroupWaves];
    extern __shared__ int exp_lds[];
    const int keys = a.p.n_experts + 2;
    uint32_t* counts = a.g + a.p.counts;
    for (int e = threadIdx.x; e < keys; e += kExpGroupThreads) {
        int s = 0;
#pragma unroll 16
        for (int c = 0; c < a.p.chunks; ++c) s += (int)counts[(size_t)c * keys + e];
        exp_lds[e] = s;
    }
    __syncthreads();
    exp_lists(a, tmp, true, [&](int e) { return exp_lds[e]; }, [&](int e, int at) {
#pragma unroll 16
        for (int c = 0; c < a.p.chunks; ++c) {
            const int n = (int)counts[(size_t)c * keys + e];
            counts[(size_t)c * keys + e] = (uint32_t)at;
            at += n;
        }
    });
}

// The rows' places.  kPlaceAlone: the one chunk of a small call, whose lists are made here too; kPlaceSum: of up to
// kExpSumChunks chunks each adds up the others' counts by itself, and the first makes the lists (a launch less: 8 us);
// kPlaceScanned: after k_expert_scan.
constexpr int kPlaceAlone = 0, kPlaceSum = 1, kPlaceScanned = 2, kExpSumChunks = 64;
template <int HOW>
__global__ __launch_bounds__(kExpGroupThreads) void k_expert_place(ExpertGroupArgs a) {
    extern __shared__ uint64_t exp_place[];           // scan; [waves][words] counts of 16 bits; [keys] starts (and totals)
    const int keys = a.p.n_experts + 2, words = (keys + 1) / 2;
    uint64_t* tmp = exp_place;
    uint32_t* hist = reinterpret_cast<uint32_t*>(tmp + kExpGroupWaves);
    int* start = reinterpret_cast<int*>(hist + kExpGroupWaves * words);
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    for (int e = threadIdx.x; e < kExpGroupWaves * words; e += kExpGroupThreads) hist[e] = 0;
    int key[kExpWaveSteps];
    exp_read_keys(a, blockIdx.x, key);
    if constexpr (HOW == kPlaceSum) {
        int* sum = start + keys;
        const uint32_t* counts = a.g + a.p.counts;
        for (int e = threadIdx.x; e < keys; e += kExpGroupThreads) {
            int all = 0, before = 0;
#pragma unroll 16
            for (int c = 0; c < a.p.chunks; ++c) {
                const int n = (int)counts[(size_t)c * keys + e];
                all += n;
                before += c < (int)blockIdx.x ? n : 0;
            }
            sum[e] = all;
            start[e] = before;
        }
        __syncthreads();
        exp_lists(a, tmp, blockIdx.x == 0, [&](int e) { return sum[e]; }, [&](int e, int at) { start[e] += at; });
    } else if constexpr (HOW == kPlaceScanned) {
        for (int e = threadIdx.x; e < keys; e += kExpGroupThreads) start[e] = (int)a.g[a.p.counts + (size_t)blockIdx.x * keys + e];
    }
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
        if constexpr (HOW == kPlaceAlone) {
            start[2 * w] = (int)(sum & 0xFFFFu);
            if (2 * w + 1 < keys) start[2 * w + 1] = (int)(sum >> 16);
        }
    }
    __syncthreads();
    if constexpr (HOW == kPlaceAlone) {
        exp_lists(a, tmp, true, [&](int e) { return start[e]; }, [&](int e, int at) { start[e] = at; });
        __syncthreads();
    }
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

// At most 64 rows (decode): a lane has a row, and learns of the others from their lanes; every wave the same, each for its
// share of the keys' first positions, the first wave for the rest.  No counts, no scans: 4 us where the general form takes 8.
constexpr int kExpFewGroup = 64;
__global__ __launch_bounds__(256) void k_expert_group_few(ExpertGroupArgs a) {
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, E = a.p.n_experts;
    const bool some = lane < a.p.n_rows;
    const int key = some ? exp_key(a, lane) : E + 2;
    for (int e = threadIdx.x; e < E + 2; e += 256) {
        int at = 0;
        for (int j = 0; j < a.p.n_rows; ++j) at += __builtin_amdgcn_readlane(key, j) < e ? 1 : 0;
        a.g[a.p.off + e] = at;
    }
    if (wave) return;
    // rows before this one's key and with it; a key's first row writes its tiles (rows of a key: at most 64, one tile and
    // up to four small ones)
    int at = 0, before = 0, rows = 0, bad = 0;
    for (int j = 0; j < a.p.n_rows; ++j) {
        const int k = __builtin_amdgcn_readlane(key, j);
        at += k < key ? 1 : 0;
        rows += k == key ? 1 : 0;
        before += k == key && j < lane ? 1 : 0;
        bad |= k == E + 1;
    }
    static_assert(kExpFewGroup <= kExpTile, "a key's rows are one tile");
    const bool leads = some && before == 0;
    int s = 0, t = 0, small = 0, tiles = 0;
    for (int j = 0; j < a.p.n_rows; ++j) {
        if (!__builtin_amdgcn_readlane(leads ? 1 : 0, j)) continue;
        const int k = __builtin_amdgcn_readlane(key, j), n = exp_tiles(__builtin_amdgcn_readlane(rows, j), kExpSmall);
        small += n;
        ++tiles;
        s += k < key ? n : 0;
        t += k < key ? 1 : 0;
    }
    if (some) a.g[a.p.order + at + before] = (uint32_t)lane;
    if (leads) {
        const int who = key < E ? key : E - 1 - key;
        if (a.p.max_small)
            for (int o = 0; o < rows; o += kExpSmall) reinterpret_cast<int4*>(a.g + a.p.small)[s++] = make_int4(who, at + o, min(kExpSmall, rows - o), 0);
        reinterpret_cast<int4*>(a.g + a.p.tiles)[t] = make_int4(who, at, rows, 0);
        reinterpret_cast<int4*>(a.g + a.p.large)[t] = make_int4(who, at, rows, 0);
    }
    if (lane == 0) {
        exp_head(a, a.p.max_small ? small : 0, tiles, tiles);
        if (bad) *reinterpret_cast<volatile unsigned int*>(a.err) = kErrExpertId;
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

// a tile, the same for all lanes: what depends on it branches as one
__device__ inline int4 exp_item(const ExpertArgs& a, size_t list, int i) {
    const int4 it = reinterpret_cast<const int4*>(a.g + list)[i];
    return make_int4(__builtin_amdgcn_readfirstlane(it.x), __builtin_amdgcn_readfirstlane(it.y), __builtin_amdgcn_readfirstlane(it.z), 0);
}
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
    work = __builtin_amdgcn_readfirstlane((id & 7) * each + q);
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

// Rows at any alignment and of any length.  A tile of BM x BN outputs, four waves of (BM / 2) x (BN / 2), the summed axis in steps of
// 128 bytes (4,096 tokens, top-8 of 128, 2,047 -> 767 in bf16: 315 us, where k_expert_fast takes 192 for one column more).
// All loads of a stage are under way before any of them is looked at: with chunks completed as they were loaded gradients took 2.5 times as long.
//   forward: rows of x by rows of W;  dx: rows of dy by columns of W;  dw: columns of dy by columns of x, summed over a
//   group's rows.
// An operand whose summed axis is contiguous in memory lies in LDS as rows of 128 bytes, its 16-byte chunks
// permuted by the row's bits (the 16 lanes that are read at once then lie in all 64 banks); one whose summed axis is
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

    static __device__ inline int at_contiguous(int row, int chunk) { return row * 128 + ((chunk ^ ((row >> 1) & 7)) << 4); }
    static __device__ inline int at_strided(int row, int chunk) {
        return row * (128 * ES) + ((ES == 2 ? chunk ^ ((row & 3) << 2) : chunk ^ ((row & 4) << 1)) << 4);
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
            for (int j = 0; j < 4; ++j) {
                const int col = c0 + (lane & 31);
                v[j] = *reinterpret_cast<const float*>(t + at_strided(s * 8 + (lane >> 5) * 4 + j, col >> 2) + (col & 3) * ES);
            }
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
        first = __builtin_amdgcn_readfirstlane(a.g[a.p.off + expert]);
        count = __builtin_amdgcn_readfirstlane(a.g[a.p.off + expert + 1]) - first;
        if (count == 0 && a.add) return;
    } else {
        if (!exp_work(blockIdx.x, (int)a.g[kExpHeadTiles] * col_tiles, work)) return;
        const int4 it = exp_item(a, a.p.tiles, work / col_tiles);
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
            pa[i] = MODE == kModeForward ? exp_row_x(a, row) : exp_row_dy(a, row);
        }
    }
    if constexpr (MODE == kModeForward) {
#pragma unroll
        for (int i = 0; i < NL; ++i) pb[i] = w + (size_t)min(n0 + rc + 32 * i, a.rows - 1) * a.k * ES;
    }
    xu4 ra[NL], rb[NL];
    // f(row, column, width): a chunk, as it is loaded
    auto load_by = [&](int k0, auto f) {
#pragma unroll
        for (int i = 0; i < NL; ++i) {
            if constexpr (MODE != kModeDw) ra[i] = f(pa[i], k0 + cc * VEC, K);
            if constexpr (MODE == kModeForward) rb[i] = f(pb[i], k0 + cc * VEC, K);
            if constexpr (MODE == kModeDx) rb[i] = f(w + (size_t)min(k0 + rs + RPI * i, K - 1) * a.k * ES, n0 + cs * VEC, a.k);
            if constexpr (MODE == kModeDw) {
                const int r = k0 + rs + RPI * i;
                const uint32_t row = order[r < K ? r : 0];
                ra[i] = f(exp_row_dy(a, row), m0 + cs * VEC, a.rows);
                rb[i] = f(exp_row_x(a, row), n0 + cs * VEC, a.k);
            }
        }
    };
    const bool narrow = min(a.k, a.rows) < VEC;             // rows shorter than a load go value by value
    auto load = [&](int k0) {
        if (narrow)
            load_by(k0, [](const uint8_t* row, int c, int width) { return exp_load<X>(row + (size_t)c * ES, width - c); });
        else
            load_by(k0, [](const uint8_t* row, int c, int width) { return exp_last<X>(row, c, width); });
    };
    // what lies past a row's end, or past the sum's rows, becomes zeros on the way to LDS, when all loads are under way
    const int over_a = narrow ? 0 : exp_over<X>(m0 + cs * VEC, a.rows), over_b = narrow ? 0 : exp_over<X>(n0 + cs * VEC, a.k);
    auto stage = [&](int buf, int k0) {
        uint8_t* ta = exp_tile + buf * 2 * G::kSide;
        uint8_t* tb = ta + G::kSide;
        const int over_k = narrow ? 0 : exp_over<X>(k0 + cc * VEC, K);
#pragma unroll
        for (int i = 0; i < NL; ++i) {
            const int past = k0 + rs + RPI * i < K ? 0 : 16;
            *reinterpret_cast<xu4*>(ta + (G::TA ? G::at_strided(rs + RPI * i, cs) : G::at_contiguous(rc + 32 * i, cc))) =
                exp_shift(ra[i], G::TA ? max(over_a, past) : over_k);
            *reinterpret_cast<xu4*>(tb + (G::TB ? G::at_strided(rs + RPI * i, cs) : G::at_contiguous(rc + 32 * i, cc))) =
                exp_shift(rb[i], G::TB ? max(over_b, past) : over_k);
        }
    };
    const int wm = (wave >> 1) * 64, wn = (wave & 1) * 64;
    xf16 acc[2][2] = {};
    const int steps = (K + BK - 1) / BK;
    if (steps) {
        load(0);
        stage(0, 0);
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
        if (t + 1 < steps) stage((t + 1) & 1, (t + 1) * BK);
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

// Where every row of every operand begins at a multiple of 16 bytes and has a whole number of them:
// both operands go from memory straight into LDS (1 KB a wave and instruction, no registers), the next stage's while the
// matrix cores run on this one.  A lane's 16 bytes land at its own place of that KB, so the permutations of ExpGemm are made
// by what each lane asks for.  Chunks past the summed axis come from `exp_zeros`; columns past the width
// repeat the first and are not stored.
// C: BM x BN tile, WM x WN waves, KB bytes of a contiguous row (or as many strided rows) a stage.
static __device__ const uint32_t exp_zeros[4] = {0u, 0u, 0u, 0u};

__device__ inline void exp_dma(const uint8_t* src, uint8_t* lds) {     // lds: the wave's; lane i fills lds + 16 i
    __builtin_amdgcn_global_load_lds((__attribute__((address_space(1))) void*)(src),
                                     (__attribute__((address_space(3))) void*)(lds), 16, 0, 0);
}
// All but the last N of a wave's transfers are done, and its LDS reads, and that holds for all waves
template <int N>
__device__ inline void exp_stage_barrier() {
    static_assert(N < 64, "vmcnt has 6 bits");
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(N) : "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// what may pass a transfer in the schedule: all but products and memory (LDS reads may)
constexpr int kSchedBetween = 0x186;
template <typename X, int MODE, int BM_, int BN_, int WM_, int WN_, int KB_, int S_>
struct ExpFast {
    static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_, KB = KB_, S = S_, NW = WM * WN, ES = (int)sizeof(typename X::S);
    static constexpr int VEC = X::kVec, BK = KB / ES, STEPS = BK / (2 * VEC);          // of a stage
    static constexpr bool TA = MODE == kModeDw, TB = MODE != kModeForward;
    static constexpr int kA = BM * KB, kB = BN * KB;                                    // bytes of a stage (BK rows of BM values as well)
    static constexpr int TRA = kA / 1024, NT = (kA + kB) / 1024 / NW;                   // transfers of A; of a wave
    static constexpr int TM = BM / WM / 32, TN = BN / WN / 32;
    static constexpr int kStages = S * (kA + kB);
    static constexpr int kWindow = 512;                    // rows of a weight gradient whose places are in LDS at a time
    static constexpr int kLds = kStages + (MODE == kModeDw ? kWindow * 16 : 0);
    static constexpr bool kLarge = BM == kExpLarge;
    static_assert(MODE == kModeDw || BM == kExpTile || BM == kExpLarge, "one of the lists' tiles");
    static_assert((kA + kB) % (1024 * NW) == 0, "whole transfers");
    static_assert(NW % 2 == 0 && TRA % 2 == 0, "a lane's transfers are whole 16 rows apart, which the permutation repeats after");

    // the chunk that lies at place p of a row, or the place of chunk p: the 16 lanes that are read at once (32 of 8
    // bytes, 64 of 4) then lie in all 64 banks
    static __device__ inline int swap_contiguous(int row, int p) { return KB == 128 ? p ^ ((row >> 1) & 7) : p ^ ((row >> 2) & 3); }
    template <int COLS>
    static __device__ inline int swap_strided(int row, int p) {
        return ES == 4 ? p ^ ((row & 4) << 1) : COLS == 64 ? p ^ ((row & 2) << 1) : p ^ ((row & 3) << 2);
    }
    static __device__ inline xu4 contiguous(const uint8_t* t, int r0, int s) {
        const int lane = threadIdx.x & 63, row = r0 + (lane & 31);
        return *reinterpret_cast<const xu4*>(t + row * KB + (swap_contiguous(row, 2 * s + (lane >> 5)) << 4));
    }
    template <int COLS>
    static __device__ inline xu4 strided(const uint8_t* t, int c0, int s) {
        const int lane = threadIdx.x & 63;
        xu4 r;
        if constexpr (ES == 2) {
            const int l = lane & 15, row = s * 16 + (lane >> 5) * 8 + (l >> 2), col = c0 + (lane & 16) + (l & 3) * 4;
            const uint8_t* p = t + row * (COLS * ES) + (swap_strided<COLS>(row, col >> 3) << 4) + ((col & 4) << 1);
            typedef __attribute__((address_space(3))) xs4 lds_xs4;
            const xs4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_xs4*)(p));
            const xs4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_xs4*)(p + 4 * COLS * ES));
            __builtin_memcpy(&r, &lo, 8);
            __builtin_memcpy(reinterpret_cast<char*>(&r) + 8, &hi, 8);
        } else {
            xf4 v;
#pragma unroll
            for (int j = 0; j < 4; ++j)
            {
                const int row = s * 8 + (lane >> 5) * 4 + j, col = c0 + (lane & 31);
                v[j] = *reinterpret_cast<const float*>(t + row * (COLS * ES) + (swap_strided<COLS>(row, col >> 2) << 4) + (col & 3) * ES);
            }
            r = __builtin_bit_cast(xu4, v);
        }
        return r;
    }
};

// The sum over `steps` stages.  Between two barriers lie the last products of a stage and the first of the next: their
// operands are in registers when the barrier is reached (the next stage's first are read right after it), so the matrix
// cores have work while the waves meet and LDS answers.  The transfers of stage t + S, into the buffer that the barrier frees,
// go between those products: issued together they hold all waves up at once.  Stages past the end are
// transferred too, as zeros: then S - 1 are always under way.  Rows: 32-row results of the wave that have rows at all.
template <typename G, typename X, int Rows, typename Transfer>
__device__ inline void exp_sum_rows(const uint8_t* tile, int steps, int wm, int wn, xf16 (&acc)[G::TM][G::TN], Transfer transfer) {
    constexpr int S = G::S, P = G::STEPS, FIRST = G::NT / P;   // transfers that follow the barrier's first products
    xu4 fa[2][G::TM], fb[2][G::TN];
    auto fragments = [&](int t, int s, int to) {
        const uint8_t* ta = tile + (t % S) * (G::kA + G::kB);
        const uint8_t* tb = ta + G::kA;
        if constexpr (Rows > 0) {
#pragma unroll
            for (int i = 0; i < Rows; ++i) {
                if constexpr (G::TA) fa[to][i] = G::template strided<G::BM>(ta, wm + 32 * i, s);
                else fa[to][i] = G::contiguous(ta, wm + 32 * i, s);
            }
#pragma unroll
            for (int j = 0; j < G::TN; ++j) {
                if constexpr (G::TB) fb[to][j] = G::template strided<G::BN>(tb, wn + 32 * j, s);
                else fb[to][j] = G::contiguous(tb, wn + 32 * j, s);
            }
        }
    };
    // the products of operands `from`, with transfers [d0, d1) of stage t among them
    auto products = [&](int from, int t, auto first, auto last) {
        constexpr int d0 = decltype(first)::value, d1 = decltype(last)::value, ALL = Rows * G::TN;
        if constexpr (Rows == 0) {
#pragma unroll
            for (int d = d0; d < d1; ++d) transfer(t, d);
        }
#pragma unroll
        for (int i = 0; i < Rows; ++i)
#pragma unroll
            for (int j = 0; j < G::TN; ++j) {
                // y and dx: the output's columns are the rows of the 32 x 32 result, so that a lane has four neighbours of them
                acc[i][j] = G::TA ? X::mma32(fa[from][i], fb[from][j], acc[i][j]) : X::mma32(fb[from][j], fa[from][i], acc[i][j]);
#pragma unroll
                for (int d = d0; d < d1; ++d)
                    if (i * G::TN + j == (d - d0) * ALL / (d1 - d0)) {
                        __builtin_amdgcn_sched_barrier(kSchedBetween);
                        transfer(t, d);
                        __builtin_amdgcn_sched_barrier(kSchedBetween);
                    }
            }
    };
    static_assert(P == 2 || P == 4, "a stage's steps");
#pragma unroll
    for (int t = 0; t < S - 1; ++t)
#pragma unroll
        for (int j = 0; j < G::NT; ++j) transfer(t, j);
    exp_stage_barrier<(S - 2) * G::NT>();
    fragments(0, 0, 0);
#pragma unroll
    for (int j = 0; j < FIRST; ++j) transfer(S - 1, j);
    for (int t = 0; t < steps; ++t) {
        fragments(t, 1, 1);
        products(0, t + S - 1, std::integral_constant<int, FIRST>{}, std::integral_constant<int, P == 2 ? G::NT : 2 * FIRST>{});
        if constexpr (P == 4) {
            fragments(t, 2, 0);
            products(1, t + S - 1, std::integral_constant<int, 2 * FIRST>{}, std::integral_constant<int, 3 * FIRST>{});
            fragments(t, 3, 1);
            products(0, t + S - 1, std::integral_constant<int, 3 * FIRST>{}, std::integral_constant<int, G::NT>{});
        }
        exp_stage_barrier<(S - 2) * G::NT>();
        fragments(t + 1, 0, 0);
        products(1, t + S, std::integral_constant<int, 0>{}, std::integral_constant<int, FIRST>{});
    }
    exp_stage_barrier<0>();                                 // nothing is under way, and the stages are free
}
template <typename G, typename X, typename Transfer>
__device__ inline void exp_sum(const uint8_t* tile, int steps, int wm, int wn, int rows, xf16 (&acc)[G::TM][G::TN], Transfer transfer) {
    if (rows > 32 * (G::TM - 1)) exp_sum_rows<G, X, G::TM>(tile, steps, wm, wn, acc, transfer);
    else if (G::TM > 2 && rows > 64) exp_sum_rows<G, X, G::TM - 1>(tile, steps, wm, wn, acc, transfer);
    else if (G::TM > 2 && rows > 32) exp_sum_rows<G, X, G::TM - 2>(tile, steps, wm, wn, acc, transfer);
    else if (rows > 0) exp_sum_rows<G, X, 1>(tile, steps, wm, wn, acc, transfer);
    else exp_sum_rows<G, X, 0>(tile, steps, wm, wn, acc, transfer);
}

// y and dx.  Transfer q of a stage fills its KB q, of A and then of B: a lane's 16 bytes come from src[j] + stage * step[j]
// while their place on the summed axis, stage * BK + at[j], is inside, and else from exp_zeros.
template <typename X, int MODE, int BM, int BN, int WM, int WN, int KB, int S, int OCC>
__global__ __launch_bounds__(64 * WM * WN, OCC) void k_expert_fast(ExpertArgs a) {
    typedef ExpFast<X, MODE, BM, BN, WM, WN, KB, S> G;
    constexpr int ES = G::ES, VEC = G::VEC, BK = G::BK, NT = G::NT;
    extern __shared__ __align__(16) uint8_t exp_tile[];
    if (!exp_groups_fit(a)) return;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int width = MODE == kModeForward ? a.rows : a.k, K = MODE == kModeForward ? a.k : a.rows;
    const int col_tiles = (width + BN - 1) / BN;
    int work;
    if (!exp_work(blockIdx.x, (int)a.g[G::kLarge ? kExpHeadLarge : kExpHeadTiles] * col_tiles, work)) return;
    const int4 it = exp_item(a, G::kLarge ? a.p.large : a.p.tiles, work / col_tiles);
    const int n0 = work % col_tiles * BN;
    if (it.x < 0) {
        exp_fill<X>(a, it, n0, BN, width);
        return;
    }
    const uint32_t* order = a.g + a.p.order + it.y;
    const uint8_t* w = a.w + (size_t)it.x * a.rows * a.k * ES;
    constexpr int RC = 1024 / KB, CC = KB / 16;             // of a contiguous operand's transfer: rows, chunks of a row
    constexpr int CB = BN * ES / 16, RB = 64 / CB;          // of a strided one's
    uint64_t src[NT], step[NT];
    int at[NT];
#pragma unroll
    for (int j = 0; j < NT; ++j) {
        const int q = j * G::NW + wave, b = q - G::TRA;
        if (q < G::TRA) {                                   // rows past the tile repeat its last and are not stored
            const int m = q * RC + lane / CC;
            const uint32_t row = order[min(m, it.z - 1)];
            at[j] = G::swap_contiguous(m, lane % CC) * VEC;
            src[j] = (uint64_t)((MODE == kModeForward ? exp_row_x(a, row) : exp_row_dy(a, row)) + at[j] * ES);
            step[j] = KB;
        } else if constexpr (!G::TB) {
            const int n = b * RC + lane / CC;
            at[j] = G::swap_contiguous(n, lane % CC) * VEC;
            src[j] = (uint64_t)(w + ((size_t)min(n0 + n, a.rows - 1) * a.k + at[j]) * ES);
            step[j] = KB;
        } else {
            const int r = b * RB + lane / CB, c = n0 + G::template swap_strided<BN>(r, lane % CB) * VEC;
            at[j] = r;
            src[j] = (uint64_t)(w + ((size_t)r * a.k + (c < a.k ? c : 0)) * ES);
            step[j] = (uint64_t)BK * a.k * ES;
        }
    }
    const int wm = wave / WN * (BM / WM), wn = wave % WN * (BN / WN);
    uint32_t out[G::TM];                                    // rows of the lane's results
#pragma unroll
    for (int i = 0; i < G::TM; ++i) out[i] = order[min(wm + 32 * i + (lane & 31), it.z - 1)];
    const uint8_t* zeros = reinterpret_cast<const uint8_t*>(exp_zeros);
    xf16 acc[G::TM][G::TN] = {};
    exp_sum<G, X>(exp_tile, (K + BK - 1) / BK, wm, wn, it.z - wm, acc, [&](int t, int j) {
        const uint8_t* p = reinterpret_cast<const uint8_t*>(src[j] + (uint64_t)t * step[j]);
        exp_dma(t * BK + at[j] < K ? p : zeros, exp_tile + (t % S) * (G::kA + G::kB) + (j * G::NW + wave) * 1024);
    });
    // a lane has output row lane % 32, columns 8 (v / 4) + 4 (lane / 32) + v % 4
#pragma unroll
    for (int i = 0; i < G::TM; ++i) {
        if (wm + 32 * i + (lane & 31) >= it.z) continue;
        uint8_t* o = exp_row_out(a, out[i]);
#pragma unroll
        for (int j = 0; j < G::TN; ++j)
#pragma unroll
            for (int v = 0; v < 16; v += 4) {
                const int n = n0 + wn + 32 * j + 2 * v + 4 * (lane >> 5);
                typename X::S s4[4];
#pragma unroll
                for (int c = 0; c < 4; ++c) s4[c] = X::put(acc[i][j][v + c]);
                if (n < width) {                            // whole fours: rows are multiples of 16 bytes
                    if constexpr (ES == 4) *reinterpret_cast<xu4*>(o + (size_t)n * ES) = __builtin_bit_cast(xu4, s4);
                    else *reinterpret_cast<xu2*>(o + (size_t)n * ES) = __builtin_bit_cast(xu2, s4);
                }
            }
    }
}

// dW: a tile of dy's columns by x's, summed over the rows of its expert.  Where the rows lie is kept in LDS, a window of them at a time.
template <typename X, int BM, int BN, int WM, int WN, int KB, int S, int OCC>
__global__ __launch_bounds__(64 * WM * WN, OCC) void k_expert_dw(ExpertArgs a) {
    typedef ExpFast<X, kModeDw, BM, BN, WM, WN, KB, S> G;
    constexpr int ES = G::ES, VEC = G::VEC, BK = G::BK, NT = G::NT;
    extern __shared__ __align__(16) uint8_t exp_tile[];
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
    const int row_tiles = (a.rows + BM - 1) / BM, col_tiles = (a.k + BN - 1) / BN;
    int work;
    if (!exp_work(blockIdx.x, a.p.n_experts * row_tiles * col_tiles, work)) return;
    const int expert = work / (row_tiles * col_tiles);
    work -= expert * row_tiles * col_tiles;
    const int m0 = work / col_tiles * BM, n0 = work % col_tiles * BN;
    // read beside the head, not after it
    const int first = __builtin_amdgcn_readfirstlane(a.g[a.p.off + expert]);
    const int count = __builtin_amdgcn_readfirstlane(a.g[a.p.off + expert + 1]) - first;
    if (!exp_groups_fit(a)) return;
    if (count == 0 && a.add) return;
    const uint32_t* order = a.g + a.p.order + first;
    constexpr int CA = BM * ES / 16, RA = 64 / CA, CB = BN * ES / 16, RB = 64 / CB;   // of a transfer: chunks of a row, rows
    int src[NT], at[NT];                                    // bytes from a row's start, row of the stage
    uint64_t* places = reinterpret_cast<uint64_t*>(exp_tile + G::kStages);   // of dy's and x's rows
#pragma unroll
    for (int j = 0; j < NT; ++j) {
        const int q = j * G::NW + wave, b = q - G::TRA;
        at[j] = q < G::TRA ? q * RA + lane / CA : b * RB + lane / CB;
        const int c = q < G::TRA ? m0 + G::template swap_strided<BM>(at[j], lane % CA) * VEC : n0 + G::template swap_strided<BN>(at[j], lane % CB) * VEC;
        src[j] = c < (q < G::TRA ? a.rows : a.k) ? c * ES : 0;
    }
    const uint8_t* zeros = reinterpret_cast<const uint8_t*>(exp_zeros);
    int to = 0;
    auto transfer = [&](int t, int j) {
        const int q = j * G::NW + wave, r = t * BK + at[j];
        const uint8_t* p = reinterpret_cast<const uint8_t*>(places[2 * (r < to ? r : 0) + (q < G::TRA ? 0 : 1)]) + src[j];
        exp_dma(r < to ? p : zeros, exp_tile + (t % S) * (G::kA + G::kB) + q * 1024);
    };
    const int wm = wave / WN * (BM / WM), wn = wave % WN * (BN / WN);
    xf16 acc[G::TM][G::TN] = {};
    for (int from = 0; from < count; from += G::kWindow) {
        to = min(count - from, G::kWindow);
        for (int r = tid; r < to; r += 64 * G::NW) {
            const uint32_t row = order[from + r];
            places[2 * r] = (uint64_t)exp_row_dy(a, row);
            places[2 * r + 1] = (uint64_t)exp_row_x(a, row);
        }
        __syncthreads();
        const int steps = (to + BK - 1) / BK;
#pragma unroll
        for (int t = 0; t < S - 1; ++t)
#pragma unroll
            for (int j = 0; j < NT; ++j) transfer(t, j);
        for (int t = 0; t < steps; ++t) {                   // stages past the end are zeros: S - 1 are always under way
            exp_stage_barrier<(S - 2) * NT>();
#pragma unroll
            for (int j = 0; j < NT; ++j) transfer(t + S - 1, j);
            const uint8_t* ta = exp_tile + (t % S) * (G::kA + G::kB);
#pragma unroll
            for (int s = 0; s < G::STEPS; ++s) {
                xu4 fa[G::TM], fb[G::TN];
#pragma unroll
                for (int i = 0; i < G::TM; ++i) fa[i] = G::template strided<BM>(ta, wm + 32 * i, s);
#pragma unroll
                for (int j = 0; j < G::TN; ++j) fb[j] = G::template strided<BN>(ta + G::kA, wn + 32 * j, s);
#pragma unroll
                for (int i = 0; i < G::TM; ++i)
#pragma unroll
                    for (int j = 0; j < G::TN; ++j) acc[i][j] = X::mma32(fa[i], fb[j], acc[i][j]);
            }
        }
        exp_stage_barrier<0>();                             // nothing is under way, and the stages are free
    }
    // of a 32 x 32 result a lane has column lane % 32 and rows 8 (v / 4) + 4 (lane / 32) + v % 4
    float* dw = a.dw + (size_t)expert * a.rows * a.k;
#pragma unroll
    for (int i = 0; i < G::TM; ++i)
#pragma unroll
        for (int j = 0; j < G::TN; ++j) {
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
}

// Few rows: a workgroup has up to 16 rows of one expert and NT * 16 rows of its W; its NW waves share k (8 where each then has
// four loads of 64 bytes a row to make at once, k of 1,024 values of 16 bits; 4 below: one token at 768 -> 2,048 9.4 us against
// 10.3, 64 tokens 225 against 249; at 2,048 -> 768 8.1 with 8, 8.6 with 4).  W's rows go
// from memory into MFMA operands (a lane has 16 bytes of row lane % 16), x's rows likewise from L2; the waves' sums meet
// in LDS, added in the waves' order.
template <typename X, int NT, int NW>
__global__ __launch_bounds__(64 * NW) void k_expert_rows(ExpertArgs a) {
    constexpr int ES = (int)sizeof(typename X::S), VEC = X::kVec, COLS = 16 * NT, STEP = 4 * VEC, U = 4;
    __shared__ xf4 part[NW][NT][64];
    if (!exp_groups_fit(a)) return;
    const int col_tiles = (a.rows + COLS - 1) / COLS;
    int work;
    if (!exp_work(blockIdx.x, (int)a.g[kExpHeadSmall] * col_tiles, work)) return;
    const int4 it = exp_item(a, a.p.small, work / col_tiles);
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
    const int steps = (a.k + STEP - 1) / STEP, each = (steps + NW - 1) / NW;
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
    for (int c = threadIdx.x; c < NT * 64; c += 64 * NW) {
        const int t = c >> 6, l = c & 63;
        xf4 v = part[0][t][l];
#pragma unroll
        for (int w = 1; w < NW; ++w) v += part[w][t][l];
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
