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
//   the sums of p stay in registers (f32) and the counts in LDS; one partial per workgroup.
// k_balance_sum:  the partials of 64 experts per workgroup, in a fixed order (no
//   float atomics: the same inputs give the same bits); the last workgroup adds up the losses.
// k_route_backward: the same split; the row stays in registers between the softmax
//   and the gradient, so the logits are read once and their gradient is written once.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace sabah {

constexpr int kBalanceThreads = 256;          // of k_balance_sum, and where a row is one wave's or four's
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
    unsigned* ticket;
    int* counts;                  // [n_groups][n_experts]
    float* mean_p;                // [n_groups][n_experts]
    float* losses;                // [2]
    int* n_valid;                 // [n_groups + 2]
    unsigned int* err;
};

// A token's row is held by W waves: one up to 512 experts, else 4 or 8, the workgroup;
// thread v of them has the experts v, v + 64 W, ....  Sums and maxima over the
// row; tmp: W floats of LDS, used with W > 1, where the whole workgroup takes part.
template <int W, typename F>
__device__ inline float row_reduce(float v, float* tmp, F f) {
#pragma unroll
    for (int k = 1; k < 64; k <<= 1) v = f(v, __shfl_xor(v, k));
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

// The softmax of a row: e becomes p.  Returns false for a row of minus infinities only.
template <int PER, int W>
__device__ inline bool row_softmax(float (&e)[PER], float& lse, float* tmp) {
    float m = -__builtin_inff(), some = 0.0f;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        m = fmaxf(m, e[j]);
        some = e[j] == -__builtin_inff() ? some : 1.0f;    // a NaN counts: it is passed on, not hidden
    }
    if (row_max<W>(some, tmp) == 0.0f) return false;
    m = row_max<W>(m, tmp);
    float s = 0.0f;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        e[j] = expf(e[j] - m);                              // 0 past the experts (row_load's minus infinities)
        s += e[j];
    }
    s = row_sum<W>(s, tmp);
    const float inv = 1.0f / s;
#pragma unroll
    for (int j = 0; j < PER; ++j) e[j] *= inv;
    lse = m + logf(s);
    return true;
}

template <int PER, int W>
__device__ inline void row_load(const uint8_t* row, int n_experts, int v, float (&e)[PER]) {
    const float* l = reinterpret_cast<const float*>(row);
#pragma unroll
    for (int j = 0; j < PER; ++j) e[j] = v + 64 * W * j < n_experts ? l[v + 64 * W * j] : -__builtin_inff();
}

// dynamic LDS: n_experts floats, n_experts ints
template <int PER, int W>
__global__ __launch_bounds__(row_threads(W)) void k_balance_rows(BalanceArgs a) {
    extern __shared__ float blds[];
    constexpr int kThr = row_threads(W), kSide = kThr / (64 * W);   // kSide tokens side by side
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
#pragma unroll
    for (int j = 0; j < PER; ++j) acc[j] = 0.0f;
    float z = 0.0f;
    int n = 0;
    const int end = min(a.group_len, (c + 1) * a.chunk_len);
    for (int i = c * a.chunk_len + side; i < end; i += kSide) {
        const size_t t = (size_t)g * a.group_len + i;
        if (a.mask && !a.mask[t]) continue;                 // with W > 1 the same for the whole workgroup
        float e[PER], lse;
        row_load<PER, W>(a.logits + t * a.stride, E, v, e);
        if (!row_softmax<PER, W>(e, lse, s_tmp)) continue;
#pragma unroll
        for (int j = 0; j < PER; ++j) acc[j] += e[j];
        z += lse * lse;
        ++n;
        if (v < a.n_used) {
            const int id = a.ids[t * a.n_used + v];
            if (id >= 0 && id < E) atomicAdd(&s_c[id], 1);
            else *reinterpret_cast<volatile unsigned int*>(a.err) = kErrRouteId;
        }
    }
    if (v == 0) {
        s_n[side] = n;
        s_z[side] = z;
    }
    // the sums of the tokens side by side, in their order
    for (int w = 0; w < kSide; ++w) {
        if (side == w) {
#pragma unroll
            for (int j = 0; j < PER; ++j) {
                const int i = v + 64 * W * j;
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

// sum over the workgroup's threads, in a fixed order; every thread gets it
template <typename T>
__device__ inline T block_sum(T v, T* tmp) {
#pragma unroll
    for (int k = 1; k < 64; k <<= 1) v += __shfl_xor(v, k);
    __syncthreads();
    if ((threadIdx.x & 63u) == 0) tmp[threadIdx.x >> 6] = v;
    __syncthreads();
    T s = tmp[0];
    for (int w = 1; w < (int)(blockDim.x >> 6); ++w) s += tmp[w];
    return s;
}

__global__ __launch_bounds__(kBalanceThreads) void k_balance_sum(BalanceArgs a) {
    constexpr int kWaves = kBalanceThreads / 64;
    __shared__ double s_d[kWaves][64];
    __shared__ int s_c[kWaves][64];
    __shared__ double s_t[kWaves];
    __shared__ int s_i[kWaves];
    __shared__ unsigned s_last;
    const int tid = (int)threadIdx.x, v = tid & 63, wave = tid >> 6, E = a.n_experts;
    const int g = (int)blockIdx.y, e = (int)blockIdx.x * 64 + v;
    const size_t p0 = (size_t)g * a.chunks;
    int n = 0;
    for (int c = tid; c < a.chunks; c += kBalanceThreads) n += __float_as_int(a.part_z[p0 + c].x);
    n = block_sum(n, s_i);
    double p = 0.0;
    int cnt = 0;
    if (e < E)
        for (int c = wave; c < a.chunks; c += kWaves) {
            p += (double)a.part_p[(p0 + c) * E + e];
            cnt += a.part_c[(p0 + c) * E + e];
        }
    s_d[wave][v] = p;
    s_c[wave][v] = cnt;
    __syncthreads();
    double term = 0.0;
    if (wave == 0 && e < E) {
        for (int w = 1; w < kWaves; ++w) p += s_d[w][v], cnt += s_c[w][v];
        const double mp = n > 0 ? p / (double)n : 0.0;
        a.counts[(size_t)g * E + e] = cnt;
        a.mean_p[(size_t)g * E + e] = (float)mp;
        if (n > 0) term = mp * (double)cnt / ((double)n * (double)a.n_used) * (double)E;
    }
    const double sum = block_sum(term, s_t);
    if (tid == 0) {
        if (blockIdx.x == 0) a.n_valid[g] = n;
        __hip_atomic_store(&a.part_loss[(size_t)g * gridDim.x + blockIdx.x], sum, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        s_last = __hip_atomic_fetch_add(a.ticket, 1u, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    if (s_last != gridDim.x * gridDim.y - 1u) return;
    // the last workgroup: every other's sums are in memory
    double loss = 0.0, z = 0.0;
    int total = 0, filled = 0;
    for (int i = tid; i < (int)(gridDim.x * gridDim.y); i += kBalanceThreads)
        loss += __hip_atomic_load(&a.part_loss[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    for (int q = tid; q < a.n_groups; q += kBalanceThreads) {
        int m = 0;
        for (int c = 0; c < a.chunks; ++c) {
            const float2 pz = a.part_z[(size_t)q * a.chunks + c];
            m += __float_as_int(pz.x);
            z += (double)pz.y;
        }
        total += m;
        filled += m > 0;
    }
    loss = block_sum(loss, s_t);
    z = block_sum(z, s_t);
    total = block_sum(total, s_i);
    filled = block_sum(filled, s_i);
    if (tid == 0) {
        a.losses[0] = filled ? (float)(loss / (double)filled) : 0.0f;
        a.losses[1] = total ? (float)(z / (double)total) : 0.0f;
        a.n_valid[a.n_groups] = total;
        a.n_valid[a.n_groups + 1] = filled;
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

template <int PER, int W>
__global__ __launch_bounds__(row_threads(W)) void k_route_backward(RouteBackArgs a) {
    __shared__ float s_tmp[W];
    const int tid = (int)threadIdx.x, v = tid % (64 * W), E = a.n_experts;
    const int t = (int)blockIdx.x * (row_threads(W) / (64 * W)) + tid / (64 * W);
    if (t >= a.n_tokens) return;                            // W = 1: whole waves leave, and no barrier follows
    float* out = reinterpret_cast<float*>(a.dlogits + (size_t)t * a.dstride);
    float p[PER], d[PER], lse = 0.0f;
    bool live = !(a.mask && !a.mask[t]);
    if (live) {
        row_load<PER, W>(a.logits + (size_t)t * a.stride, E, v, p);
        live = row_softmax<PER, W>(p, lse, s_tmp);
    }
#pragma unroll
    for (int j = 0; j < PER; ++j) d[j] = 0.0f;
    if (live && a.counts) {
        const int g = t / a.group_len;
        const float n_g = (float)a.n_valid[g], n = (float)a.n_valid[a.n_groups], filled = (float)a.n_valid[a.n_groups + 1];
        const float cb = a.c_balance * (float)E / (n_g * filled), fs = 1.0f / (n_g * (float)a.n_used);
        const float cz = 2.0f * a.c_z * lse / n;
        float dot = 0.0f;
#pragma unroll
        for (int j = 0; j < PER; ++j)
            if (v + 64 * W * j < E) {
                d[j] = (float)a.counts[(size_t)g * E + v + 64 * W * j] * fs;
                dot += d[j] * p[j];
            }
        dot = row_sum<W>(dot, s_tmp);
#pragma unroll
        for (int j = 0; j < PER; ++j) d[j] = p[j] * (cb * (d[j] - dot) + cz);
    }
    if (live && a.dw) {
        int id = -1;
        float w = 0.0f, l = -__builtin_inff();
        const int slot = v & 63;                            // every wave of the row holds the slots
        if (slot < a.n_used) {
            id = a.ids[(size_t)t * a.n_used + slot];
            w = a.dw[(size_t)t * a.n_used + slot];
            if (id < 0 || id >= E) {
                *reinterpret_cast<volatile unsigned int*>(a.err) = kErrRouteId;
                id = -1;
                w = __builtin_nanf("");                     // the row becomes NaN
            } else {
                l = reinterpret_cast<const float*>(a.logits + (size_t)t * a.stride)[id];
            }
        }
        // the selected experts' shares, lane j with slot j
        const float m = a.norm_w ? row_max<1>(l, s_tmp) : lse;
        float q = slot < a.n_used && l > -__builtin_inff() ? expf(l - m) : 0.0f;
        if (l != l) q = l;
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
        for (int k = 0; k < a.n_used; ++k) {                // in slot order: an expert named twice gets both
            const int ik = __builtin_amdgcn_readlane(id, k);
            const float ak = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(add), k));
#pragma unroll
            for (int j = 0; j < PER; ++j)
                if (v + 64 * W * j == ik) d[j] += ak;
        }
    }
#pragma unroll
    for (int j = 0; j < PER; ++j)
        if (v + 64 * W * j < E) out[v + 64 * W * j] = d[j];
}

}  // namespace sabah
