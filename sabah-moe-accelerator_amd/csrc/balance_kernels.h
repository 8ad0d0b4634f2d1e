// The router's training losses and the gradient of its logits, beside
// k_route's gating (route_kernels.h).
//
//   p_t = softmax(l_t), lse_t = log sum exp l_t, over the valid tokens (mask) of
//   n_groups groups of equal length (the sequences of a padded batch, or one group)
//   counts_ge = valid (token, slot) pairs of group g with expert e,  n_g its valid tokens
//   mean_p_ge = (1 / n_g) sum p_te,  f_ge = counts_ge / (n_g n_used)
//   losses[0] = mean over the groups with a valid token of  E sum_e f_ge mean_p_ge
//   losses[1] = (1 / n) sum lse_t^2
// A row of minus infinities only has no distribution: its token counts as masked.
//
// k_balance_rows: one wave per token at a time (a workgroup above 512 experts), a workgroup per run of a group's tokens;
//   the sums of p stay in registers (f32 for 64 tokens at a time, those sums in 64 bits: the 8,192 tokens that a lane
//   of a long batch has would be off by 1e-4 in f32) and the counts in LDS; one partial per workgroup.
// k_balance_sum:  the partials of 16 experts per workgroup, in a fixed order (no
//   float atomics: the same inputs give the same bits); the last workgroup adds up the losses.
// k_route_backward: the same split; the row stays in registers between the softmax
//   and the gradient, so the logits are read once and their gradient is written once.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

namespace sabah {

constexpr int kBalanceThreads = 256;          // where a row is one wave's or four's
constexpr int kBalanceSumThreads = 1024, kBalanceCols = 16;   // of k_balance_sum, and its experts per workgroup
constexpr int row_threads(int w) { return w > 4 ? 64 * w : kBalanceThreads; }
constexpr unsigned kErrRouteId = 3u;          // sticky error word: a selected expert id out of range

struct BalanceArgs {
    const uint8_t* logits;        // [n_tokens] rows of n_experts floats, `stride` bytes apart
    size_t stride;
    const int32_t* ids;           // [n_tokens][n_used]
    const uint8_t* mask;          // [n_tokens], 0: masked; null: every token valid
    int n_experts, n_used, n_groups, group_len;
    int chunks, chunk_len;        // a group's tokens in `chunks` runs of chunk_len
    float* part_p;                // [n_groups * chunks][n_experts]
    int* part_c;                  // the same of counts
    float2* part_z;               // [n_groups * chunks] (valid tokens' number as int bits, sum of lse^2)
    double* part_loss;            // [n_groups * column blocks]
    double2* group;               // [n_groups] (valid tokens, sum of lse^2)
    unsigned* ticket;
    int* counts;                  // [n_groups][n_experts]
    float* mean_p;                // [n_groups][n_experts]
    float* losses;                // [2]
    int* n_valid;                 // [n_groups + 2]
    unsigned int* err;
};

// A token's row is held by W waves: one up to 512 experts, else 4 or 8, the workgroup.  Thread v of them
// has VEC neighbours of every 64 W VEC experts, PER in all.
template <int VEC, int W>
__device__ inline int row_expert(int v, int j) { return 64 * W * VEC * (j / VEC) + VEC * v + j % VEC; }

// Sums and maxima over the row, the same bits in every lane: within 16 lanes by DPP, then across them
// by lane swaps (shuffles through LDS took a token's three reductions from 0.1 to 0.6 us).
// tmp: W floats of LDS, used with W > 1, where the whole workgroup takes part.
template <int CTRL>
__device__ inline float row_dpp(float v) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xF, 0xF, false));
}
template <int W, typename F>
__device__ inline float row_reduce(float v, float* tmp, F f) {
    v = f(v, row_dpp<0xB1>(v));                             // quad_perm [1,0,3,2]
    v = f(v, row_dpp<0x4E>(v));                             // quad_perm [2,3,0,1]
    v = f(v, row_dpp<0x141>(v));                            // row_half_mirror
    v = f(v, row_dpp<0x140>(v));                            // row_mirror
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = f(__uint_as_float(r[0]), __uint_as_float(r[1]));
    const auto h = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = f(__uint_as_float(h[0]), __uint_as_float(h[1]));
    if constexpr (W > 1) {
        __syncthreads();
        if ((threadIdx.x & 63u) == 0) tmp[threadIdx.x >> 6] = v;
        __syncthreads();
        v = tmp[0];
#pragma unroll
        for (int w = 1; w < W; ++w) v = f(v, tmp[w]);
    }
    return v;
}
template <int W>
__device__ inline float row_max(float v, float* tmp) {
    return row_reduce<W>(v, tmp, [](float a, float b) { return fmaxf(a, b); });
}
template <int W>
__device__ inline float row_sum(float v, float* tmp) {
    return row_reduce<W>(v, tmp, [](float a, float b) { return a + b; });
}

// exp(x) as 2^(x log2 e), with the rest that the product's rounding and log2 e's own leave out as a factor 1 + rest ln 2
__device__ inline float row_exp(float x) {
    constexpr float kLog2e = 1.44269502162933349609375f, kLog2eRest = 1.92596299e-8f, kLn2 = 0.693147182f;
    const float t = x * kLog2e, rest = __builtin_fmaf(x, kLog2eRest, __builtin_fmaf(x, kLog2e, -t));
    const float e = __builtin_amdgcn_exp2f(t);
    return t > -126.0f && t < 126.0f ? __builtin_fmaf(e, rest * kLn2, e) : e;   // past them e is 0 or infinite, and x may be
}

// The softmax of a row: e becomes p; m, inv: the row's largest logit, and p is exp(l - m) inv.  Returns false for a row of
// minus infinities only.
template <int PER, int W>
__device__ inline bool row_softmax(float (&e)[PER], float& m, float& inv, float& lse, float* tmp) {
    m = -__builtin_inff();
    bool nan = false;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        m = fmaxf(m, e[j]);
        nan |= e[j] != e[j];                                // passed on, not hidden
    }
    if (nan) m = __builtin_inff();                          // every difference is then a NaN or an infinity: the row becomes NaN
    m = row_max<W>(m, tmp);
    if (m == -__builtin_inff()) return false;
    float s = 0.0f;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        e[j] = row_exp(e[j] - m);                           // 0 past the experts (row_load's minus infinities)
        s += e[j];
    }
    s = row_sum<W>(s, tmp);
    inv = m == __builtin_inff() ? __builtin_nanf("") : 1.0f / s;
#pragma unroll
    for (int j = 0; j < PER; ++j) e[j] *= inv;
    lse = m + logf(s);
    if (m == __builtin_inff()) lse = row_max<W>(nan ? 1.0f : 0.0f, tmp) > 0.0f ? __builtin_nanf("") : m;   // m: an infinite logit
    return true;
}

typedef float rf4 __attribute__((ext_vector_type(4), aligned(4)));
typedef float rf2 __attribute__((ext_vector_type(2), aligned(4)));
typedef int ri4 __attribute__((ext_vector_type(4), aligned(4)));
typedef int ri2 __attribute__((ext_vector_type(2), aligned(4)));

// T: float or int, of one row; `past` beyond the experts
template <int PER, int VEC, int W, typename T>
__device__ inline void row_load(const void* row, int n_experts, int v, T past, T (&e)[PER]) {
    typedef typename std::conditional<std::is_same<T, int>::value, ri4, rf4>::type T4;
    typedef typename std::conditional<std::is_same<T, int>::value, ri2, rf2>::type T2;
    const T* l = static_cast<const T*>(row);
#pragma unroll
    for (int j = 0; j < PER; j += VEC) {
        const int i = row_expert<VEC, W>(v, j);
        if (i + VEC <= n_experts) {
            if constexpr (VEC == 4) {
                const T4 w = *reinterpret_cast<const T4*>(l + i);
#pragma unroll
                for (int c = 0; c < 4; ++c) e[j + c] = w[c];
            } else if constexpr (VEC == 2) {
                const T2 w = *reinterpret_cast<const T2*>(l + i);
                e[j] = w[0], e[j + 1] = w[1];
            } else {
                e[j] = l[i];
            }
        } else {
#pragma unroll
            for (int c = 0; c < VEC; ++c) e[j + c] = i + c < n_experts ? l[i + c] : past;
        }
    }
}

// dynamic LDS: n_experts floats, n_experts ints
template <int PER, int VEC, int W>
__global__ __launch_bounds__(row_threads(W)) void k_balance_rows(BalanceArgs a) {
    extern __shared__ float blds[];
    constexpr int kThr = row_threads(W), kSide = kThr / (64 * W);   // kSide tokens side by side
    constexpr int B = W == 1 ? 4 : 1;                       // and B of them loaded at a time
    constexpr int kRun = 64;                                // terms summed in f32; such sums meet in 64 bits
    __shared__ int s_n[kSide];
    __shared__ float s_z[kSide];
    __shared__ float s_tmp[W];
    float* s_p = blds;
    int* s_c = reinterpret_cast<int*>(blds + a.n_experts);
    const int tid = (int)threadIdx.x, v = tid % (64 * W), side = tid / (64 * W), E = a.n_experts;
    const int g = (int)blockIdx.y, c = (int)blockIdx.x;
    const size_t part = (size_t)g * a.chunks + c;
    if (tid == 0 && part == 0) *a.ticket = 0u;              // k_balance_sum's, which the next launch reads
    for (int i = tid; i < E; i += kThr) s_c[i] = 0;
    __syncthreads();
    float acc[PER];
    double sum[PER], z_sum = 0.0;
#pragma unroll
    for (int j = 0; j < PER; ++j) acc[j] = 0.0f, sum[j] = 0.0;
    float z = 0.0f;
    int n = 0, left = kRun / B;
    const int end = min(a.group_len, (c + 1) * a.chunk_len);
    for (int i0 = c * a.chunk_len + side; i0 < end; i0 += kSide * B) {
        float e[B][PER];
        int id[B];
        bool live[B];
#pragma unroll
        for (int b = 0; b < B; ++b) {
            const int i = min(i0 + kSide * b, end - 1);     // past the run: a token again, which counts nothing
            const size_t t = (size_t)g * a.group_len + i;
            live[b] = i0 + kSide * b < end && !(a.mask && !a.mask[t]);   // the same for all threads of the row
            if (!live[b]) continue;
            row_load<PER, VEC, W>(a.logits + t * a.stride, E, v, -__builtin_inff(), e[b]);
            id[b] = v < a.n_used ? a.ids[t * a.n_used + v] : 0;
        }
#pragma unroll
        for (int b = 0; b < B; ++b) {
            float m, inv, lse;
            if (!live[b] || !row_softmax<PER, W>(e[b], m, inv, lse, s_tmp)) continue;
#pragma unroll
            for (int j = 0; j < PER; ++j) acc[j] += e[b][j];
            z += lse * lse;
            ++n;
            if (v < a.n_used) {
                if (id[b] >= 0 && id[b] < E) atomicAdd(&s_c[id[b]], 1);
                else *reinterpret_cast<volatile unsigned int*>(a.err) = kErrRouteId;
            }
        }
        if (--left == 0) {
            left = kRun / B;
#pragma unroll
            for (int j = 0; j < PER; ++j) sum[j] += (double)acc[j], acc[j] = 0.0f;
            z_sum += (double)z, z = 0.0f;
        }
    }
#pragma unroll
    for (int j = 0; j < PER; ++j) acc[j] = (float)(sum[j] + (double)acc[j]);
    if (v == 0) {
        s_n[side] = n;
        s_z[side] = (float)(z_sum + (double)z);
    }
    // the sums of the tokens side by side, in their order
    for (int w = 0; w < kSide; ++w) {
        if (side == w) {
#pragma unroll
            for (int j = 0; j < PER; ++j) {
                const int i = row_expert<VEC, W>(v, j);
                if (i < E) s_p[i] = w ? s_p[i] + acc[j] : acc[j];
            }
        }
        __syncthreads();
    }
    for (int i = tid; i < E; i += kThr) {
        a.part_p[part * E + i] = s_p[i];
        a.part_c[part * E + i] = s_c[i];
    }
    if (tid == 0) {
        int nn = 0;
        float zz = 0.0f;
        for (int w = 0; w < kSide; ++w) nn += s_n[w], zz += s_z[w];
        a.part_z[part] = make_float2(__int_as_float(nn), zz);
    }
}

// sum over a wave, in a fixed order; every lane gets it
template <typename T>
__device__ inline T wave_add(T v) {
#pragma unroll
    for (int k = 1; k < 64; k <<= 1) v += __shfl_xor(v, k);
    return v;
}

// Thread (chunk row, expert): 64 rows of the chunks by 16 experts.  grid (16s of experts, groups)
__global__ __launch_bounds__(kBalanceSumThreads) void k_balance_sum(BalanceArgs a) {
    constexpr int kWaves = kBalanceSumThreads / 64, U = 8;
    __shared__ double s_p[kWaves][kBalanceCols], s_z[kWaves];
    __shared__ int s_c[kWaves][kBalanceCols], s_n[kWaves];
    const int tid = (int)threadIdx.x, lane = tid & 63, wave = tid >> 6, E = a.n_experts;
    const int g = (int)blockIdx.y, e = (int)blockIdx.x * kBalanceCols + (tid & 15), r0 = tid >> 4;
    const size_t p0 = (size_t)g * a.chunks;
    double p = 0.0, z = 0.0;
    int cnt = 0, n = 0;
    for (int c0 = r0; c0 < a.chunks; c0 += 64 * U) {        // U loads at a time
        float x[U];
        int k[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const size_t at = (p0 + min(c0 + 64 * u, a.chunks - 1)) * E + min(e, E - 1);
            x[u] = a.part_p[at];
            k[u] = a.part_c[at];
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (c0 + 64 * u < a.chunks) {
                p += (double)x[u];
                cnt += k[u];
            }
    }
    for (int c = tid; c < a.chunks; c += kBalanceSumThreads) {
        const float2 pz = a.part_z[p0 + c];
        n += __float_as_int(pz.x);
        z += (double)pz.y;
    }
    p += __shfl_xor(p, 16);
    p += __shfl_xor(p, 32);
    cnt += __shfl_xor(cnt, 16);
    cnt += __shfl_xor(cnt, 32);
    n = wave_add(n);
    z = wave_add(z);
    if (lane < kBalanceCols) {
        s_p[wave][lane] = p;
        s_c[wave][lane] = cnt;
    }
    if (lane == 0) {
        s_n[wave] = n;
        s_z[wave] = z;
    }
    __syncthreads();
    if (wave != 0) return;
    n = 0, z = 0.0, p = 0.0, cnt = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) n += s_n[w], z += s_z[w], p += s_p[w][lane & 15], cnt += s_c[w][lane & 15];
    double term = 0.0;
    if (lane < kBalanceCols && e < E) {
        const double mp = n > 0 ? p / (double)n : 0.0;
        a.counts[(size_t)g * E + e] = cnt;
        a.mean_p[(size_t)g * E + e] = (float)mp;
        if (n > 0) term = mp * (double)cnt / ((double)n * (double)a.n_used) * (double)E;
    }
    term = wave_add(term);
    // the last workgroup to come adds up the groups: what the others wrote for it they wrote past their caches
    unsigned last = 0u;
    if (lane == 0) {
        if (blockIdx.x == 0) {
            a.n_valid[g] = n;
            __hip_atomic_store(&a.group[g].x, (double)n, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            __hip_atomic_store(&a.group[g].y, z, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
        __hip_atomic_store(&a.part_loss[(size_t)g * gridDim.x + blockIdx.x], term, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        last = __hip_atomic_fetch_add(a.ticket, 1u, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT);
    }
    last = (unsigned)__builtin_amdgcn_readfirstlane((int)last);
    if (last != gridDim.x * gridDim.y - 1u) return;
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "agent");
    double loss = 0.0, total = 0.0, filled = 0.0;
    z = 0.0;
    for (int i = lane; i < (int)(gridDim.x * gridDim.y); i += 64)
        loss += __hip_atomic_load(&a.part_loss[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    for (int q = lane; q < a.n_groups; q += 64) {
        const double m = __hip_atomic_load(&a.group[q].x, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        z += __hip_atomic_load(&a.group[q].y, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        total += m;
        filled += m > 0.0 ? 1.0 : 0.0;
    }
    loss = wave_add(loss);
    z = wave_add(z);
    total = wave_add(total);
    filled = wave_add(filled);
    if (lane == 0) {
        a.losses[0] = filled > 0.0 ? (float)(loss / filled) : 0.0f;
        a.losses[1] = total > 0.0 ? (float)(z / total) : 0.0f;
        a.n_valid[a.n_groups] = (int)total;
        a.n_valid[a.n_groups + 1] = (int)filled;
    }
}

// ---------------------------------------------------------------------------
// dlogits.  With q the selected experts' share (norm_w: of their own sum, else p):
//   norm_w   dl_{id_j} += w_scale q_j (dw_j - sum_i q_i dw_i)
//   else     dl_e += w_scale p_e (sum_{j: id_j = e} dw_j - sum_j dw_j p_{id_j})
//   balance  dl_e += c_balance E / (n_g filled) p_e (f_ge - sum_i f_gi p_i)
//   z        dl_e += c_z 2 lse p_e / n
// ---------------------------------------------------------------------------
struct RouteBackArgs {
    const uint8_t* logits;
    size_t stride;
    const int32_t* ids;
    const uint8_t* mask;
    const float* dw;              // [n_tokens][n_used], or null
    const int* counts;            // [n_groups][n_experts], or null: no loss's gradient
    const int* n_valid;           // [n_groups + 2]
    uint8_t* dlogits;
    size_t dstride;
    int n_tokens, n_experts, n_used, norm_w, n_groups, group_len;
    float w_scale, c_balance, c_z;
    unsigned int* err;
};

// The selected experts' parts meet the row in LDS: a lane adds up the parts of its slot's expert in slot order
// (an expert may be named twice), the expert's first slot stores the sum, and the row's lanes pick theirs up.
template <int PER, int VEC, int W>
__global__ __launch_bounds__(row_threads(W)) void k_route_backward(RouteBackArgs a) {
    constexpr int kSide = row_threads(W) / (64 * W);
    __shared__ float s_tmp[W];
    __shared__ float s_add[kSide][64 * W * PER];
    const int tid = (int)threadIdx.x, v = tid % (64 * W), side = tid / (64 * W), slot = tid & 63, E = a.n_experts;
    const int t = ((int)blockIdx.y * (int)gridDim.x + (int)blockIdx.x) * kSide + side;
    if (t >= a.n_tokens) return;                            // W = 1: whole waves leave, and no barrier follows
    const uint8_t* row = a.logits + (size_t)t * a.stride;
    float* out = reinterpret_cast<float*>(a.dlogits + (size_t)t * a.dstride);
    float p[PER], d[PER], top = 0.0f, inv = 0.0f, lse = 0.0f;
    int counts[PER], id = -1;
    float w = 0.0f, l = -__builtin_inff(), n_g = 0.0f, n = 0.0f, filled = 0.0f;
    bool live = !(a.mask && !a.mask[t]), bad = false;
    if (live) {                                             // every load before the first result is needed
        row_load<PER, VEC, W>(row, E, v, -__builtin_inff(), p);
        if (a.dw && slot < a.n_used) {
            id = a.ids[(size_t)t * a.n_used + slot];
            w = a.dw[(size_t)t * a.n_used + slot];
        }
        if (a.counts) {
            const int g = t / a.group_len;
            row_load<PER, VEC, W>(a.counts + (size_t)g * E, E, v, 0, counts);
            n_g = (float)a.n_valid[g], n = (float)a.n_valid[a.n_groups], filled = (float)a.n_valid[a.n_groups + 1];
        }
        if (a.dw && slot < a.n_used) {
            bad = id < 0 || id >= E;
            if (bad) {
                w = __builtin_nanf("");                     // the row becomes NaN
                id = -1;
            } else {
                l = reinterpret_cast<const float*>(row)[id];
            }
        }
        live = row_softmax<PER, W>(p, top, inv, lse, s_tmp);
        // k_route has no expert for a row of minus infinities and names -1: no error, its token counts as masked
        if (live && bad) *reinterpret_cast<volatile unsigned int*>(a.err) = kErrRouteId;
    }
#pragma unroll
    for (int j = 0; j < PER; ++j) d[j] = 0.0f;
    if (live && a.counts) {
        const float cb = a.c_balance * (float)E / (n_g * filled), fs = 1.0f / (n_g * (float)a.n_used);
        const float cz = 2.0f * a.c_z * lse / n;
        float dot = 0.0f;
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            d[j] = (float)counts[j] * fs;
            dot += d[j] * p[j];
        }
        dot = row_sum<W>(dot, s_tmp);
#pragma unroll
        for (int j = 0; j < PER; ++j) d[j] = p[j] * (cb * (d[j] - dot) + cz);
    }
    if (live && a.dw) {
        // the selected experts' shares, lane j with slot j (every wave of the row holds the slots)
        const float m = a.norm_w ? row_max<1>(l, s_tmp) : top;
        float q = slot < a.n_used && l > -__builtin_inff() ? row_exp(l - m) : 0.0f;
        if (l != l) q = l;
        if (!a.norm_w) q *= inv;
        if (a.norm_w) {
            const float s = row_sum<1>(q, s_tmp);
            q = s > 0.0f || s != s ? q / s : 0.0f;
        }
        const float dot = row_sum<1>(q * w, s_tmp);
        const float add = a.w_scale * q * (a.norm_w ? w - dot : w);
        if (!a.norm_w || dot != dot) {
#pragma unroll
            for (int j = 0; j < PER; ++j) d[j] -= a.w_scale * p[j] * dot;
        }
        float sum = 0.0f;
        bool first = id >= 0;
        for (int k = 0; k < a.n_used; ++k) {
            const bool same = __builtin_amdgcn_readlane(id, k) == id;
            const float ak = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(add), k));
            sum += same ? ak : 0.0f;
            first = first && !(same && k < slot);
        }
        float* mine = s_add[side];
#pragma unroll
        for (int j = 0; j < PER; ++j) mine[row_expert<VEC, W>(v, j)] = 0.0f;
        if constexpr (W > 1) __syncthreads();
        __builtin_amdgcn_wave_barrier();
        if (first && tid % (64 * W) < 64) mine[id] = sum;
        if constexpr (W > 1) __syncthreads();
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int j = 0; j < PER; ++j) d[j] += mine[row_expert<VEC, W>(v, j)];
    }
    // The wide rows are streamed past the caches: 11.9 us against 13.4 (16,384 tokens of 512 experts), no difference at 512 tokens
#pragma unroll
    for (int j = 0; j < PER; j += VEC) {
        const int i = row_expert<VEC, W>(v, j);
        if (i + VEC <= E) {
            if constexpr (VEC == 4) __builtin_nontemporal_store(rf4{d[j], d[j + 1], d[j + 2], d[j + 3]}, reinterpret_cast<rf4*>(out + i));
            else if constexpr (VEC == 2) *reinterpret_cast<rf2*>(out + i) = rf2{d[j], d[j + 1]};
            else out[i] = d[j];
        } else {
#pragma unroll
            for (int c = 0; c < VEC; ++c)
                if (i + c < E) out[i + c] = d[j + c];
        }
    }
}

}  // namespace sabah
