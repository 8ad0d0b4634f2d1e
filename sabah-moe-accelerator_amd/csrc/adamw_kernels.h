// An AdamW step over many tensors at once.
//   g = c * grad, c = grad_scale * min(1, max_norm / (norm + 1e-6)), norm = grad_scale * |all gradients|
//   m = b1 m + (1 - b1) g;  v = b2 v + (1 - b2) g^2;  p = p (1 - lr decay) - lr / (1 - b1^t) * m / (sqrt(v / (1 - b2^t)) + eps)
// Moments are kept in 32 bits, or in 8 bits with a 32-bit scale, the largest value, for each block of 256:
//   m: sign * (code / 127)^2 * scale;  v: (code / 255)^4 * scale
// even steps of m's square root and v's fourth root (of sqrt(v)'s square root, sqrt(v) being what divides m): steps next to
// the block's largest are 1.6 %, and values down to 6e-5 (m) and 2.4e-10 (v) of it are told from 0.  A v above 0 never
// becomes 0: the division by sqrt(v) would blow its m up.  A code is the nearest one, found in 64 bits: next to
// the border of two codes an error of 32 bits would be a whole step.  What the nearest code cannot say is lost in each step: with
// b2 = 0.999 a v below its block's largest decays with the block's scale alone (a step of 0.1 %, half a code is 0.8 % at least), and
// only squares of many times v raise it.  So v comes out too large over some thousand steps: 1.1 times after 2,000 of even
// noise, 1.4 after 5,000 (single blocks 2.5); 45 times where all but one gradient of a block became a tenth.
// UNBIASED codes take the lower or the upper of the two codes around a value in proportion to where it lies between them, so
// that moments are right in the mean at any b1 and b2 (both: an m that the nearest code holds up would be divided by a v that
// goes on falling), with a noise of at most sqrt(2 / code) of v, 9 % near the block's largest.  The choice is a hash of the step's
// number and the value's place, so that a state and a gradient give the same bits again (302 M values in bf16 with master
// copies: 1,374 us, 1,098 with the nearest codes).
//
// k_adamw_norm:  the gradients' sum of squares in 64 bits, by a fixed number of workgroups, in a fixed order.
// k_adamw_begin: the norm, the step's number and what depends on them, by one workgroup (of one wave where no norm is wanted).
// k_adamw_step:  2,048 values of one tensor to a workgroup; every state is read and written once, which bounds it: 604 M values
//   in f32 3,180 us, 5.3 TB/s; 302 M in bf16 with master copies and 8-bit moments 1,098 us, 4.9 TB/s (1,430 with f32's
//   correctly rounded roots and division, which the 64-bit codes do not need: they are found by their borders).
#pragma once
#include "balance_kernels.h"   // row_max
#include "expert_kernels.h"    // storage types

namespace sabah {

constexpr int kAdamBlock = 256, kAdamChunk = 2048, kAdamThreads = 256;
constexpr int kAdamNormGroups = 1024;
constexpr float kAdamMost = 3.4028234663852886e38f;  // f32's largest number

// A tensor as the device sees it; m and v begin at `at` of the flat moments, a multiple of kAdamBlock
struct AdamTensor {
    uint8_t* p;
    const uint8_t* g;
    float* master;                 // or null
    double decay;
    long long n, at;
    int p_type, g_type;            // 0, 1, 30
};
struct AdamChunk {
    int tensor;
    int first;                     // in chunks
};
// What k_adamw_begin leaves for k_adamw_step
struct AdamScalars {
    double c;
    float rate, root;              // lr / (1 - b1^t), 1 / sqrt(1 - b2^t)
    double lr;
    int skip, pad;
    uint64_t draw;                 // of the step, for unbiased codes
};
struct AdamArgs {
    const AdamTensor* tensors;
    const AdamChunk* chunks;
    int n_chunks, bits;
    void *m, *v;                   // float or codes
    float *m_scale, *v_scale;
    double b1, b2, eps, lr, grad_scale, max_norm;
    const float* lr_dev;           // or null: lr
    long long* step;
    float* norm;                   // or null
    double* part;                  // [kAdamNormGroups]
    int parts;
    AdamScalars* s;
};

template <typename X>
__device__ inline void adam_load4(const uint8_t* p, long long i, int left, float (&e)[4]) {
    const typename X::S* q = reinterpret_cast<const typename X::S*>(p) + i;
    if (left >= 4) {
        typename X::S s[4];
        if constexpr (X::kVec == 4) {
            const xu4 w = *reinterpret_cast<const xu4u*>(q);
            __builtin_memcpy(s, &w, 16);
        } else {
            const xu2 w = *reinterpret_cast<const xu2u*>(q);
            __builtin_memcpy(s, &w, 8);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) e[j] = (float)s[j];
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) e[j] = j < left ? (float)q[j] : 0.0f;
    }
}
template <typename X>
__device__ inline void adam_store4(uint8_t* p, long long i, int left, const float (&e)[4]) {
    typename X::S* q = reinterpret_cast<typename X::S*>(p) + i;
    if (left >= 4) {
        typename X::S s[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) s[j] = X::put(e[j]);
        if constexpr (X::kVec == 4) {
            xu4 w;
            __builtin_memcpy(&w, s, 16);
            *reinterpret_cast<xu4u*>(q) = w;
        } else {
            xu2 w;
            __builtin_memcpy(&w, s, 8);
            *reinterpret_cast<xu2u*>(q) = w;
        }
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (j < left) q[j] = X::put(e[j]);
    }
}
__device__ inline void adam_load(int type, const uint8_t* p, long long i, int left, float (&e)[4]) {
    if (type == 0) adam_load4<ExpF32>(p, i, left, e);
    else if (type == 1) adam_load4<ExpF16>(p, i, left, e);
    else adam_load4<ExpBF16>(p, i, left, e);
}
__device__ inline void adam_store(int type, uint8_t* p, long long i, int left, const float (&e)[4]) {
    if (type == 0) adam_store4<ExpF32>(p, i, left, e);
    else if (type == 1) adam_store4<ExpF16>(p, i, left, e);
    else adam_store4<ExpBF16>(p, i, left, e);
}

__device__ inline double adam_block_sum(double v, double* tmp) {
    const int wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
#pragma unroll
    for (int d = 32; d; d >>= 1) v += __shfl_xor(v, d);
    if ((threadIdx.x & 63) == 0) tmp[wave] = v;
    __syncthreads();
    v = tmp[0];
    for (int w = 1; w < waves; ++w) v += tmp[w];
    return v;
}

__global__ __launch_bounds__(kAdamThreads) void k_adamw_norm(AdamArgs a) {
    __shared__ double tmp[kAdamThreads / 64];
    double s = 0.0;
    for (int c = blockIdx.x; c < a.n_chunks; c += gridDim.x) {
        const AdamChunk ch = a.chunks[c];
        const AdamTensor T = a.tensors[ch.tensor];
        const long long at = (long long)ch.first * kAdamChunk;
        float g[kAdamChunk / kAdamThreads / 4][4];
#pragma unroll
        for (int k = 0; k < kAdamChunk / kAdamThreads / 4; ++k) {
            const long long i = at + (k * kAdamThreads + (int)threadIdx.x) * 4;
            adam_load(T.g_type, T.g, i, (int)min(4ll, T.n - i), g[k]);
        }
#pragma unroll
        for (int k = 0; k < kAdamChunk / kAdamThreads / 4; ++k)
#pragma unroll
            for (int j = 0; j < 4; ++j) s = __builtin_fma((double)g[k][j], (double)g[k][j], s);
    }
    s = adam_block_sum(s, tmp);
    if (threadIdx.x == 0) a.part[blockIdx.x] = s;
}

// 64 bits of a number: the SplitMix64 generator's output after it (Steele, Lea and Flood, 2014)
__device__ inline uint64_t adam_mix(uint64_t z) {
    z += 0x9E3779B97F4A7C15ull;
    z = (z ^ (z >> 30)) * 0xBF58476D1CE4E5B9ull;
    z = (z ^ (z >> 27)) * 0x94D049BB133111EBull;
    return z ^ (z >> 31);
}

__global__ __launch_bounds__(1024) void k_adamw_begin(AdamArgs a) {
    __shared__ double tmp[16];
    // the powers of both betas at once, in two lanes, while the sums arrive
    const long long t = *a.step + 1;
    const double lr = a.lr_dev ? (double)*a.lr_dev : a.lr;
    double s = a.norm && (int)threadIdx.x < a.parts ? a.part[threadIdx.x] : 0.0, c = a.grad_scale, rest = 0.0;
    if (threadIdx.x < 64) rest = 1.0 - pow(threadIdx.x & 1 ? a.b2 : a.b1, (double)t);
    const double rest2 = __shfl(rest, 1);
    bool skip = false;
    if (a.norm) {                                           // uniform
        s = adam_block_sum(s, tmp);
        const double norm = sqrt(s) * a.grad_scale;
        skip = !(norm < __builtin_inf());                   // an infinite or NaN gradient: nothing changes
        c *= fmin(1.0, a.max_norm / (norm + 1e-6));
        if (threadIdx.x == 0) *a.norm = skip ? (float)norm : fminf(kAdamMost, (float)norm);   // infinite or NaN: not made
    }
    if (threadIdx.x == 0) {
        AdamScalars r{};
        r.c = c;
        r.lr = lr;
        r.rate = (float)(lr / rest);
        r.root = (float)(1.0 / sqrt(rest2));
        r.skip = skip;
        r.draw = adam_mix((uint64_t)t);
        *a.s = r;
        if (!skip) *a.step = t;
    }
}

// The nearest code to t = (code)^2 (m's), to t = (code)^4 (v's): f32's root, then its neighbours' borders in 64 bits
__device__ inline int adam_code2(double t, int most) {
    int k = min(most, (int)rintf(__builtin_amdgcn_sqrtf((float)t)));   // off by at most one, which the borders mend
    const double k2 = (double)(k * k) + 0.25;               // (k +- 1/2)^2 = k^2 +- k + 1/4
    if (t > k2 + (double)k) ++k;
    else if (t < k2 - (double)k) --k;
    return min(most, max(0, k));
}
__device__ inline int adam_code4(double t, int most) {
    int k = min(most, (int)rintf(__builtin_amdgcn_sqrtf(__builtin_amdgcn_sqrtf((float)t))));
    const double k2 = (double)(k * k) + 0.25, hi = k2 + (double)k, lo = k2 - (double)k;
    if (t > hi * hi) ++k;
    else if (k > 0 && t < lo * lo) --k;
    return min(most, max(0, k));
}
// The code below t, or the one above where `bits` of 32, as a share of the way to it, lie before t
__device__ inline int adam_either(double t, double lo, double hi, int k, uint32_t bits) {
    return ((double)bits + 0.5) * 0x1p-32 * (hi - lo) < t - lo ? k + 1 : k;
}
__device__ inline int adam_either2(double t, int most, uint32_t bits) {
    int k = min(most - 1, (int)__builtin_amdgcn_sqrtf((float)t));
    if (t < (double)(k * k)) --k;                           // f32's root is off by at most one
    else if (k + 1 < most && t >= (double)((k + 1) * (k + 1))) ++k;
    return adam_either(t, (double)(k * k), (double)((k + 1) * (k + 1)), k, bits);
}
__device__ inline int adam_either4(double t, int most, uint32_t bits) {
    auto fourth = [](int k) { return (double)(k * k) * (double)(k * k); };
    int k = min(most - 1, (int)__builtin_amdgcn_sqrtf(__builtin_amdgcn_sqrtf((float)t)));
    if (t < fourth(k)) --k;
    else if (k + 1 < most && t >= fourth(k + 1)) ++k;
    return adam_either(t, fourth(k), fourth(k + 1), k, bits);
}
constexpr double kAdamM2 = 127.0 * 127.0, kAdamV4 = 255.0 * 255.0 * 255.0 * 255.0;

// Four neighbours a lane, a block of 256 a wave: the codes and the scales of m and v
__device__ inline float adam_block_max(float v) {
    v = row_max<1>(v, nullptr);
    return v;
}
// at: the first value's place and the step's draw, of UNBIASED codes
template <bool UNBIASED>
__device__ inline void adam_encode(const double (&m)[4], const double (&v)[4], uint32_t& mc, uint32_t& vc, float& ms, float& vs,
                                   uint64_t at) {
    float hm = 0.0f, hv = 0.0f;
    bool nan = false;
#pragma unroll
    for (int j = 0; j < 4; ++j) {                           // rounding keeps the order, so the largest of the rounded is the scale
        hm = fmaxf(hm, fminf(kAdamMost, (float)fabs(m[j])));
        hv = fmaxf(hv, fminf(kAdamMost, (float)v[j]));
        nan |= m[j] != m[j] || v[j] != v[j];
    }
    hm = adam_block_max(hm);
    hv = adam_block_max(hv);
    if (__ballot(nan)) hm = hv = __builtin_nanf("");        // codes have no NaN: the block becomes it
    ms = hm;
    vs = hv;
    const double im = hm > 0.0f ? kAdamM2 / (double)hm : 0.0, iv = hv > 0.0f ? kAdamV4 / (double)hv : 0.0;
    mc = vc = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const double tm = fmin(fabs(m[j]) * im, kAdamM2), tv = fmin(v[j] * iv, kAdamV4);
        const uint64_t bits = UNBIASED ? adam_mix(at + (uint64_t)j) : 0;
        int k = UNBIASED ? adam_either2(tm, 127, (uint32_t)bits) : adam_code2(tm, 127);
        if (m[j] < 0.0) k = -k;
        mc |= (uint32_t)(k & 0xFF) << (8 * j);
        k = UNBIASED ? adam_either4(tv, 255, (uint32_t)(bits >> 32)) : adam_code4(tv, 255);
        if (k == 0 && v[j] > 0.0) k = 1;
        vc |= (uint32_t)k << (8 * j);
    }
}
__device__ inline void adam_decode(uint32_t mc, uint32_t vc, float ms, float vs, double (&m)[4], double (&v)[4]) {
    const double sm = (double)ms / kAdamM2, sv = (double)vs / kAdamV4;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int k = (int)(int8_t)(mc >> (8 * j));
        m[j] = (double)(k * (k < 0 ? -k : k)) * sm;
        const uint32_t q = (vc >> (8 * j)) & 0xFFu, q2 = q * q;
        v[j] = (double)(q2 * q2) * sv;                      // 255^4 < 2^32
    }
}

// p (1 - lost) - step, by what p loses: 1 - lost in f32 is a whole number of steps of 2^-24, for lr 1e-5 and decay 0.01 a decay
// 19 % too large.  Without decay an infinite p stays what it is.
__device__ inline float adam_move(float p, float lost, float step) { return p - ((lost != 0.0f ? p * lost : 0.0f) + step); }

// The instruction's roots, which take what lies below 2^-126 for 0: m would be divided by eps alone.  Rare enough for a branch
// of four values (302 M values: 12 us of 1,080; a branch for each takes 23, selects without one 28)
__device__ inline void adam_roots(const float (&v)[4], float (&r)[4]) {
#pragma unroll
    for (int j = 0; j < 4; ++j) r[j] = __builtin_amdgcn_sqrtf(v[j]);
    if (fminf(fminf(v[0], v[1]), fminf(v[2], v[3])) < 0x1p-126f) [[unlikely]] {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (v[j] < 0x1p-126f) r[j] = __builtin_amdgcn_sqrtf(v[j] * 0x1p64f) * 0x1p-32f;
    }
}

template <int BITS, bool UNBIASED>
__global__ __launch_bounds__(kAdamThreads) void k_adamw_step(AdamArgs a) {
    const AdamChunk ch = a.chunks[blockIdx.x];
    const AdamTensor T = a.tensors[ch.tensor];
    const AdamScalars s = *a.s;
    if (s.skip) return;
    constexpr int NK = kAdamChunk / kAdamThreads / 4;
    float g[NK][4], p[NK][4], m[NK][4], v[NK][4], ms[NK], vs[NK];
    uint32_t mc[NK], vc[NK];
    const long long first = (long long)ch.first * kAdamChunk;
#pragma unroll
    for (int k = 0; k < NK; ++k) {
        const long long i = first + (k * kAdamThreads + (int)threadIdx.x) * 4;
        const int left = (int)min(4ll, T.n - i);
        adam_load(T.g_type, T.g, i, left, g[k]);
        if (T.master) adam_load4<ExpF32>(reinterpret_cast<const uint8_t*>(T.master), i, left, p[k]);
        else adam_load(T.p_type, T.p, i, left, p[k]);
        if constexpr (BITS == 32) {
            adam_load4<ExpF32>(reinterpret_cast<const uint8_t*>(a.m), T.at + i, left, m[k]);
            adam_load4<ExpF32>(reinterpret_cast<const uint8_t*>(a.v), T.at + i, left, v[k]);
        } else if (left > 0) {                              // the flat moments fill whole blocks
            const long long b = (T.at + i) / kAdamBlock;
            mc[k] = *reinterpret_cast<const uint32_t*>(static_cast<const uint8_t*>(a.m) + T.at + i);
            vc[k] = *reinterpret_cast<const uint32_t*>(static_cast<const uint8_t*>(a.v) + T.at + i);
            ms[k] = a.m_scale[b];
            vs[k] = a.v_scale[b];
        } else {
            mc[k] = vc[k] = 0;
            ms[k] = vs[k] = 0.0f;
        }
    }
    const float lost = (float)(s.lr * T.decay), eps = (float)a.eps;
    const float b1 = (float)a.b1, n1 = (float)(1.0 - a.b1), b2 = (float)a.b2, n2 = (float)(1.0 - a.b2);
#pragma unroll
    for (int k = 0; k < NK; ++k) {
        const long long i = first + (k * kAdamThreads + (int)threadIdx.x) * 4;
        const int left = (int)min(4ll, T.n - i);
        if constexpr (BITS == 32) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float q = (float)((double)g[k][j] * s.c);   // s.c may lie outside f32's numbers
                m[k][j] = m[k][j] * b1 + q * n1;
                v[k][j] = v[k][j] * b2 + q * q * n2;
            }
            adam_store4<ExpF32>(static_cast<uint8_t*>(a.m), T.at + i, left, m[k]);
            adam_store4<ExpF32>(static_cast<uint8_t*>(a.v), T.at + i, left, v[k]);
        } else {
            double dm[4], dv[4];
            adam_decode(mc[k], vc[k], ms[k], vs[k], dm, dv);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const double q = j < left ? (double)g[k][j] * s.c : 0.0;
                dm[j] = __builtin_fma(dm[j], a.b1, q * (1.0 - a.b1));
                dv[j] = __builtin_fma(dv[j], a.b2, q * q * (1.0 - a.b2));
                m[k][j] = (float)dm[j];
                v[k][j] = (float)dv[j];
            }
            float hm, hv;
            adam_encode<UNBIASED>(dm, dv, mc[k], vc[k], hm, hv, s.draw + (uint64_t)(T.at + i));   // by whole waves
            if (left > 0) {
                *reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(a.m) + T.at + i) = mc[k];
                *reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(a.v) + T.at + i) = vc[k];
                if ((threadIdx.x & 63) == 0) {
                    a.m_scale[(T.at + i) / kAdamBlock] = hm;
                    a.v_scale[(T.at + i) / kAdamBlock] = hv;
                }
            }
        }
        float root[4];
        if constexpr (BITS == 8) adam_roots(v[k], root);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if constexpr (BITS == 32) {
                p[k][j] = adam_move(p[k][j], lost, m[k][j] / (sqrtf(v[k][j]) * s.root + eps) * s.rate);
            } else {
                // the instructions' roots and inverses, off by a step of f32: 8 bits' moments are off by 2^-7, and the step's
                // own arithmetic is what this kernel waits for.  A v that overflows f32 has an infinite root: no change
                const float r = root[j] * s.root + eps;
                p[k][j] = adam_move(p[k][j], lost, m[k][j] * __builtin_amdgcn_rcpf(r) * s.rate);
            }
        }
        if (T.master) adam_store4<ExpF32>(reinterpret_cast<uint8_t*>(T.master), i, left, p[k]);
        if (!T.master || T.p_type != 0) adam_store(T.p_type, T.p, i, left, p[k]);
    }
}

// Moments of 8 bits as the values they stand for, and values as codes: a wave per block
struct AdamMomentArgs {
    uint8_t *m_code, *v_code;
    float *m_scale, *v_scale, *m, *v;
    long long blocks;
};
__global__ __launch_bounds__(kAdamThreads) void k_adamw_decode(AdamMomentArgs a) {
    const long long b = ((long long)blockIdx.y * gridDim.x + blockIdx.x) * (kAdamThreads / 64) + (threadIdx.x >> 6);
    if (b >= a.blocks) return;
    const long long i = b * kAdamBlock + (threadIdx.x & 63) * 4;
    double m[4], v[4];
    adam_decode(*reinterpret_cast<const uint32_t*>(a.m_code + i), *reinterpret_cast<const uint32_t*>(a.v_code + i), a.m_scale[b],
                a.v_scale[b], m, v);
    const float fm[4] = {(float)m[0], (float)m[1], (float)m[2], (float)m[3]}, fv[4] = {(float)v[0], (float)v[1], (float)v[2], (float)v[3]};
    adam_store4<ExpF32>(reinterpret_cast<uint8_t*>(a.m), i, 4, fm);
    adam_store4<ExpF32>(reinterpret_cast<uint8_t*>(a.v), i, 4, fv);
}
__global__ __launch_bounds__(kAdamThreads) void k_adamw_encode(AdamMomentArgs a) {
    const long long b = ((long long)blockIdx.y * gridDim.x + blockIdx.x) * (kAdamThreads / 64) + (threadIdx.x >> 6);
    if (b >= a.blocks) return;
    const long long i = b * kAdamBlock + (threadIdx.x & 63) * 4;
    float fm[4], fv[4], ms, vs;
    adam_load4<ExpF32>(reinterpret_cast<const uint8_t*>(a.m), i, 4, fm);
    adam_load4<ExpF32>(reinterpret_cast<const uint8_t*>(a.v), i, 4, fv);
    const double m[4] = {fm[0], fm[1], fm[2], fm[3]}, v[4] = {fv[0], fv[1], fv[2], fv[3]};
    uint32_t mc, vc;
    adam_encode<false>(m, v, mc, vc, ms, vs, 0);
    *reinterpret_cast<uint32_t*>(a.m_code + i) = mc;
    *reinterpret_cast<uint32_t*>(a.v_code + i) = vc;
    if ((threadIdx.x & 63) == 0) {
        a.m_scale[b] = ms;
        a.v_scale[b] = vs;
    }
}

}  // namespace sabah
