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

struct LoraF32 { typedef float T; };
struct LoraF16 { typedef uint16_t T; };
struct LoraBF16 { typedef uint16_t T; };

__device__ inline float lora_value(LoraF32, float w) { return w; }
__device__ inline float lora_value(LoraF16, uint16_t w) { return __half2float(__ushort_as_half(w)); }
__device__ inline float lora_value(LoraBF16, uint16_t w) { return __uint_as_float((uint32_t)w << 16); }

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
        for (int i = v; i < k; i += 64) acc = __builtin_fmaf(lora_value(W{}, A[(size_t)r * k + i]), x[i], acc);
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) acc += __shfl_xor(acc, o);
        if (v == 0) s[r] = acc;
    }
    __syncthreads();
}

// one workgroup per row
template <typename W>
__global__ __launch_bounds__(kLoraThreads) void k_lora_rows(LoraArgs a) {
    __shared__ float s[kLoraMaxRank];
    const int row = (int)blockIdx.x, key = lora_key(a, row);
    float* dst = reinterpret_cast<float*>(a.dst + lora_at(row, a.n_ids, a.dst_id, a.dst_tok));
    const float* base =
        a.base ? reinterpret_cast<const float*>(a.base + lora_at(row, a.n_ids, a.base_id, a.base_tok)) : nullptr;
    if (key == kLoraBad) {
        if (threadIdx.x == 0) *reinterpret_cast<volatile unsigned int*>(a.err) = kErrLora;
        for (int o = (int)threadIdx.x; o < a.rows; o += kLoraThreads) dst[o] = __builtin_nanf("");
        return;
    }
    if (key == kLoraNone) {
        if (base != dst)
            for (int o = (int)threadIdx.x; o < a.rows; o += kLoraThreads) dst[o] = base ? base[o] : 0.0f;
        return;
    }
    const int rk = lora_rank(a, key);
    const float c = lora_scale(a, key);
    lora_shrink<W>(static_cast<const typename W::T*>(a.a) + (size_t)key * a.rank * a.k, lora_x(a, row), a.k, rk, s);
    const typename W::T* B = static_cast<const typename W::T*>(a.b) + (size_t)key * a.rows * a.rank;
    for (int o = (int)threadIdx.x; o < a.rows; o += kLoraThreads) {
        float acc = 0.0f;
        for (int r = 0; r < rk; ++r) acc = __builtin_fmaf(lora_value(W{}, B[(size_t)o * a.rank + r]), s[r], acc);
        dst[o] = base ? __builtin_fmaf(c, acc, base[o]) : c * acc;
    }
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
        for (int o = v; o < a.rows; o += 64) acc = __builtin_fmaf(lora_value(W{}, B[(size_t)o * a.rank + r]), dy[o], acc);
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
        for (int r = 0; r < rk; ++r) acc = __builtin_fmaf(lora_value(W{}, A[(size_t)r * a.k + i]), u[r], acc);
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
