// The norms around a block: after it, with the block's gate and the scale of its branch on the residual
// stream, and before the next one.  n(v; w) = v / sqrt(mean(v^2) + eps) * w, per row.
//   forward    x' = x + scale * sigmoid(gate) * n(y; w_after)  (or y itself),  h = n(x'; w_before),
//              h of x' as it is stored, so that the backward pass, which reads x' again, sees the same row
//   backward   u = x' r, r = (mean x'^2 + eps)^-1/2:  d = dout + r (w_before dh - u mean(w_before dh u)),  dx = d,
//              dw_before = sum over tokens of dh u;  with dn = scale sigmoid(gate) d the same rule gives dy and dw_after
//              from y, and dgate = sigmoid(gate) sigmoid(-gate) scale sum(d n(y)): 1 - sigmoid(gate) in f32 would have lost 6 % at a
//              gate of 16 and all of it from 17
// A row is held in registers by one wave or by a workgroup from its loads to its stores: each input is read and
// each output written once, which is what bounds it (4,001 tokens of 2,560 in bf16 forward 15.5 us, 5.3 TB/s with the
// last-level cache's help; 16,384 of 2,048 backward 92 us, 4.4 TB/s, and 6 for the weights' sums; a large copy 4.86).  8 values a
// thread: with 16 a row of 2,560 kept 4,096 places, 19.0 us, and the backward spilled.  Loading the next token's rows
// ahead changed nothing (87 us), nor did 512 or 2,048 parts (96, 84 + 13).  Sums are f32, of rounded inputs; x', h, dx and dy are rounded once.
#pragma once
#include "balance_kernels.h"   // row_reduce
#include "expert_kernels.h"    // storage types

namespace sabah {

constexpr int kNormMaxWidth = 8192;
struct NormArgs {
    const uint8_t *x, *y, *dout, *dh;      // x: forward x, backward x'
    uint8_t *out, *h, *dx, *dy;
    size_t x_st, y_st, dout_st, dh_st, out_st, h_st, dx_st, dy_st;
    const float *gate, *w_after, *w_before;
    float* dgate;
    float *part_after, *part_before;       // [parts][width]
    float scale, eps;
    int n_tokens, width, per_part;         // backward: rows of a part
};

template <typename X>
__device__ inline void norm_unpack(xu4 w, float* v) {
    typename X::S s[X::kVec];
    __builtin_memcpy(s, &w, 16);
#pragma unroll
    for (int j = 0; j < X::kVec; ++j) v[j] = (float)s[j];
}
template <typename X>
__device__ inline xu4 norm_pack(const float* v) {
    typename X::S s[X::kVec];
#pragma unroll
    for (int j = 0; j < X::kVec; ++j) s[j] = X::put(v[j]);
    xu4 w;
    __builtin_memcpy(&w, s, 16);
    return w;
}
// Thread v of a row's 64 W has kVec neighbours of every 64 W kVec columns, PER in all, kept as they were loaded (8 values
// of 16 bits in 4 registers) and widened where they are used.
template <typename X, int W>
__device__ inline int norm_col(int v, int q) { return (64 * W * q + v) * X::kVec; }

// kVec values from column c of a row, zeros past its width.  Only a row narrower than a load (NARROW: where one wave has
// it) goes value by value.
template <typename X, bool NARROW>
__device__ inline xu4 norm_chunk(const uint8_t* row, int c, int width) {
    if (NARROW && width < X::kVec) return exp_load<X>(row + (size_t)c * sizeof(typename X::S), width - c);
    return exp_chunk<X>(row, c, width);
}
template <typename X, int PER, int W>
struct NormRow {
    static constexpr int Q = PER / X::kVec;
    xu4 raw[Q];
    __device__ inline void load(const uint8_t* row, int width, int v) {
#pragma unroll
        for (int q = 0; q < Q; ++q) raw[q] = norm_chunk<X, W == 1>(row, norm_col<X, W>(v, q), width);
    }
    __device__ inline void get(int q, float (&e)[X::kVec]) const { norm_unpack<X>(raw[q], e); }
    __device__ inline void put(int q, const float (&e)[X::kVec]) { raw[q] = norm_pack<X>(e); }
    __device__ inline void store(uint8_t* row, int width, int v) const {
#pragma unroll
        for (int q = 0; q < Q; ++q) {
            const int c = norm_col<X, W>(v, q);
            exp_store<X>(row + (size_t)c * sizeof(typename X::S), raw[q], width - c);
        }
    }
};
// f32 weights at chunk q's columns (0 past the width)
template <typename X, int W>
__device__ inline void norm_weights(const float* w, int width, int v, int q, float (&e)[X::kVec]) {
#pragma unroll
    for (int j = 0; j < X::kVec; j += 4)
        norm_unpack<ExpF32>(norm_chunk<ExpF32, W == 1>(reinterpret_cast<const uint8_t*>(w), norm_col<X, W>(v, q) + j, width), &e[j]);
}
__device__ inline float norm_sigmoid(float g) { return 1.0f / (1.0f + expf(-g)); }
__device__ inline float norm_inverse(float sum_squares, int width, float eps) {
    return 1.0f / sqrtf(sum_squares / (float)width + eps);
}

constexpr int norm_threads(int w) { return w == 1 ? 256 : 64 * w; }

template <typename X, int PER, int W>
__global__ __launch_bounds__(norm_threads(W)) void k_block_norm(NormArgs a) {
    constexpr int V = X::kVec, Q = PER / V;
    __shared__ float tmp[W];
    const int v = W == 1 ? (int)threadIdx.x & 63 : (int)threadIdx.x;
    const long long group = (long long)blockIdx.y * gridDim.x + blockIdx.x, t = W == 1 ? group * 4 + (threadIdx.x >> 6) : group;
    if (t >= a.n_tokens) return;                            // W > 1: the whole workgroup
    NormRow<X, PER, W> x, y;
    float wa[PER], wb[PER], e[V], f[V];
    x.load(a.x + (size_t)t * a.x_st, a.width, v);
    if (a.y) y.load(a.y + (size_t)t * a.y_st, a.width, v);
    auto weights = [&](const float* w, float (&to)[PER]) {
#pragma unroll
        for (int q = 0; q < Q; ++q) norm_weights<X, W>(w, a.width, v, q, reinterpret_cast<float(&)[V]>(to[q * V]));
    };
    if (a.w_after) weights(a.w_after, wa);
    if (a.w_before) weights(a.w_before, wb);
    if (a.y) {
        float c = a.scale, r = 1.0f;
        if (a.gate) c *= norm_sigmoid(a.gate[t]);
        if (a.w_after) {
            float s = 0.0f;
#pragma unroll
            for (int q = 0; q < Q; ++q) {
                y.get(q, f);
#pragma unroll
                for (int j = 0; j < V; ++j) s += f[j] * f[j];
            }
            r = norm_inverse(row_sum<W>(s, tmp), a.width, a.eps);
        }
#pragma unroll
        for (int q = 0; q < Q; ++q) {
            x.get(q, e);
            y.get(q, f);
#pragma unroll
            for (int j = 0; j < V; ++j) e[j] = e[j] + c * (a.w_after ? f[j] * r * wa[q * V + j] : f[j]);
            x.put(q, e);
        }
        x.store(a.out + (size_t)t * a.out_st, a.width, v);
    }
    if (a.w_before) {
        float s = 0.0f;
#pragma unroll
        for (int q = 0; q < Q; ++q) {
            x.get(q, e);
#pragma unroll
            for (int j = 0; j < V; ++j) s += e[j] * e[j];
        }
        const float r = norm_inverse(row_sum<W>(s, tmp), a.width, a.eps);
#pragma unroll
        for (int q = 0; q < Q; ++q) {
            x.get(q, e);
#pragma unroll
            for (int j = 0; j < V; ++j) e[j] = e[j] * r * wb[q * V + j];
            x.put(q, e);
        }
        x.store(a.h + (size_t)t * a.h_st, a.width, v);
    }
}

// Backward: a part is a run of tokens of one wave (W = 1: four parts to a workgroup) or workgroup; the weights'
// gradients of its tokens stay in registers and are written as one row of partial sums.  8 values a thread: with 16 the two
// weights, their gradients and four rows take more than 200 registers.
template <typename X, int PER, int W>
__global__ __launch_bounds__(norm_threads(W)) void k_block_norm_back(NormArgs a) {
    constexpr int V = X::kVec, Q = PER / V;
    __shared__ float tmp[W];
    const int v = W == 1 ? (int)threadIdx.x & 63 : (int)threadIdx.x;
    const int part = W == 1 ? blockIdx.x * 4 + (threadIdx.x >> 6) : blockIdx.x;
    const int t0 = part * a.per_part, t1 = min(a.n_tokens, t0 + a.per_part);
    if (W == 1 && t0 >= a.n_tokens) return;
    float wa[PER], wb[PER], ga[PER] = {}, gb[PER] = {};
#pragma unroll
    for (int q = 0; q < Q; ++q) {
        if (a.w_after) norm_weights<X, W>(a.w_after, a.width, v, q, reinterpret_cast<float(&)[V]>(wa[q * V]));
        if (a.w_before) norm_weights<X, W>(a.w_before, a.width, v, q, reinterpret_cast<float(&)[V]>(wb[q * V]));
    }
    const float inv = 1.0f / (float)a.width;
    const bool read_y = a.y && a.dy && (a.w_after || a.gate);
    for (int t = t0; t < t1; ++t) {
        float d[PER], e[V], f[V];
        NormRow<X, PER, W> x, g, y, o;
        if (a.w_before) {
            x.load(a.x + (size_t)t * a.x_st, a.width, v);
            g.load(a.dh + (size_t)t * a.dh_st, a.width, v);
        }
        if (read_y) y.load(a.y + (size_t)t * a.y_st, a.width, v);
        if (a.dout) o.load(a.dout + (size_t)t * a.dout_st, a.width, v);
        if (a.dout) {
#pragma unroll
            for (int q = 0; q < Q; ++q) o.get(q, reinterpret_cast<float(&)[V]>(d[q * V]));
        } else {
#pragma unroll
            for (int j = 0; j < PER; ++j) d[j] = 0.0f;
        }
        if (a.w_before) {
            float sxx = 0.0f, sxg = 0.0f;
#pragma unroll
            for (int q = 0; q < Q; ++q) {
                x.get(q, e);
                g.get(q, f);
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    sxx += e[j] * e[j];
                    sxg += e[j] * (f[j] * wb[q * V + j]);
                }
            }
            sxx = row_sum<W>(sxx, tmp);
            sxg = row_sum<W>(sxg, tmp);
            const float r = norm_inverse(sxx, a.width, a.eps), m = sxg * r * inv;   // mean(w_before dh u)
#pragma unroll
            for (int q = 0; q < Q; ++q) {
                x.get(q, e);
                g.get(q, f);
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const float u = e[j] * r;
                    gb[q * V + j] += f[j] * u;
                    d[q * V + j] += r * (f[j] * wb[q * V + j] - u * m);
                }
                o.put(q, reinterpret_cast<float(&)[V]>(d[q * V]));
            }
            o.store(a.dx + (size_t)t * a.dx_st, a.width, v);
        }
        if (a.dy) {
            float c = a.scale, shut = 0.0f, r = 0.0f, m = 0.0f;
            if (a.gate) {
                const float g = a.gate[t], e = expf(-g), sg = 1.0f / (1.0f + e);
                c *= sg;
                shut = g > 0.0f ? e * sg : 1.0f - sg;           // sigmoid(-gate)
            }
            if (read_y) {
                float syy = 0.0f, sdy = 0.0f;
#pragma unroll
                for (int q = 0; q < Q; ++q) {
                    y.get(q, e);
#pragma unroll
                    for (int j = 0; j < V; ++j) {
                        syy += e[j] * e[j];
                        sdy += e[j] * (a.w_after ? d[q * V + j] * wa[q * V + j] : d[q * V + j]);
                    }
                }
                sdy = row_sum<W>(sdy, tmp);
                if (a.w_after) {
                    r = norm_inverse(row_sum<W>(syy, tmp), a.width, a.eps);
                    sdy *= r;                                   // sum(d n(y))
                    m = sdy * inv;
                }
                if (a.gate && v == 0) a.dgate[t] = shut * c * sdy;
            }
#pragma unroll
            for (int q = 0; q < Q; ++q) {
                if (a.w_after) y.get(q, e);
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    f[j] = c * d[q * V + j];
                    if (a.w_after) {
                        const float u = e[j] * r;
                        ga[q * V + j] += f[j] * u;
                        f[j] = c * r * (d[q * V + j] * wa[q * V + j] - u * m);
                    }
                }
                o.put(q, f);
            }
            o.store(a.dy + (size_t)t * a.dy_st, a.width, v);
        }
    }
#pragma unroll
    for (int q = 0; q < Q; ++q)
#pragma unroll
        for (int j = 0; j < V; j += 4) {
            const int c = norm_col<X, W>(v, q) + j;
            const size_t at = (size_t)part * a.width + c;
            if (a.w_after) exp_store<ExpF32>(reinterpret_cast<uint8_t*>(a.part_after + at), norm_pack<ExpF32>(&ga[q * V + j]), a.width - c);
            if (a.w_before) exp_store<ExpF32>(reinterpret_cast<uint8_t*>(a.part_before + at), norm_pack<ExpF32>(&gb[q * V + j]), a.width - c);
        }
}

// The parts' sums, 16 columns to a workgroup, in a fixed order and in 64 bits (a part's row is read in 64-byte pieces, but by
// twice the workgroups of 32 columns: 7.6 us against 11.2 for 1,024 parts of 2 x 2,048)
struct NormSumArgs {
    const float* part[2];
    float* out[2];
    int parts, width, add;
};
constexpr int kNormSumCols = 16, kNormSumLanes = 64;
__global__ __launch_bounds__(kNormSumCols * kNormSumLanes) void k_block_norm_sum(NormSumArgs a) {
    __shared__ double sums[kNormSumLanes][kNormSumCols];
    const int c = threadIdx.x % kNormSumCols, lane = threadIdx.x / kNormSumCols, col = blockIdx.x * kNormSumCols + c;
    const float* p = a.part[blockIdx.y];
    double s = 0.0;
    if (col < a.width) {
#pragma unroll 8
        for (int i = lane; i < a.parts; i += kNormSumLanes) s += (double)p[(size_t)i * a.width + col];
    }
    sums[lane][c] = s;
    __syncthreads();
    if (lane == 0 && col < a.width) {
        for (int l = 1; l < kNormSumLanes; ++l) s += sums[l][c];
        float* o = a.out[blockIdx.y] + col;
        *o = a.add ? (float)((double)*o + s) : (float)s;
    }
}

}  // namespace sabah
