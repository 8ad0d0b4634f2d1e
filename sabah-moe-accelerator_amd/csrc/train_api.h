// C-ABI entry points of a block's own weights in training: the norms around it (norm_kernels.h), its
// experts' products in float types (expert_kernels.h) and AdamW (adamw_kernels.h).  Included by sabah_rt.hip after
// adapt_api.h, whose OnDevice, align256 and type codes they use.  Device scratch is the caller's.
#pragma once

static bool float_type(int type) { return type == kTypeF32 || type == kTypeF16 || type == kTypeBF16; }
static size_t float_size(int type) { return type == kTypeF32 ? 4 : 2; }

// Memory of a tensor: n rows of `bytes`, `stride` apart (what is written may be no other tensor's memory); a row may itself be
// m parts of `part` bytes, `inner` apart
struct MemRows {
    const void* p;
    size_t stride, bytes;
    int n;
    size_t inner = 0, part = 0;
    int m = 1;
};
// Whether parts are apart as columns of one buffer are: every stride is a multiple of s, and modulo s they do not meet
static bool parts_apart(const MemRows& a, const MemRows& b, size_t off) {
    size_t s = 0;
    for (const MemRows* r : {&a, &b}) {
        if (r->n > 1) s = std::gcd(s, r->stride);
        if (r->m > 1) s = std::gcd(s, r->inner);
    }
    const size_t first = a.m > 1 ? a.part : a.bytes, second = b.m > 1 ? b.part : b.bytes;
    return s && first <= s && second <= s && off % s >= first && off % s + second <= s;
}
static bool rows_meet(const MemRows& x, const MemRows& y) {
    if (!x.p || !y.p || x.n <= 0 || y.n <= 0) return false;
    const bool swap = (uintptr_t)x.p > (uintptr_t)y.p;
    const MemRows &a = swap ? y : x, &b = swap ? x : y;
    const size_t off = (uintptr_t)b.p - (uintptr_t)a.p;
    if (off >= (size_t)(a.n - 1) * a.stride + a.bytes) return false;
    // one within the other's span: apart only as columns of rows of one length, or of their parts
    if ((a.m > 1 || b.m > 1) && parts_apart(a, b, off)) return false;
    if (a.n == 1 || b.n == 1 || a.stride != b.stride || a.bytes > a.stride || b.bytes > b.stride) return true;
    return off % a.stride < a.bytes || off % a.stride + b.bytes > a.stride;
}

// ---------------------------------------------------------------------------
// norms
// ---------------------------------------------------------------------------
// Tokens whose weight gradients one part adds up in f32, and the parts that fill the chip
constexpr int kNormPartTokens = 64, kNormParts = 768;
static void norm_plan(int n_tokens, int& parts, int& per_part) {
    per_part = std::max(1, std::min(kNormPartTokens, (n_tokens + kNormParts - 1) / kNormParts));
    parts = (n_tokens + per_part - 1) / per_part;
}

static int check_norm(const char* what, const sabah_norm_desc* n, int n_tokens) {
    if (!n) return fail("%s: null pointer", what);
    if (!float_type(n->type)) return fail("%s: type %d is none of F32 (0), F16 (1), BF16 (30)", what, n->type);
    if (n->width <= 0 || n->width > kNormMaxWidth) return fail("%s: width %d outside [1, %d]", what, n->width, kNormMaxWidth);
    if (n_tokens < 0 || n_tokens > 1 << 24) return fail("%s: n_tokens %d outside [0, %d]", what, n_tokens, 1 << 24);
    if (!(n->eps >= 0.0f) || n->eps == __builtin_inff()) return fail("%s: eps must be finite and not negative", what);
    return 0;
}
static bool norm_rows_ok(const sabah_norm_desc* n, int n_tokens, const void* p, size_t stride) {
    return !p || (stride % float_size(n->type) == 0 && (stride >= n->width * float_size(n->type) || n_tokens <= 1));
}

static MemRows norm_mem(const sabah_norm_desc* n, int n_tokens, const void* p, size_t stride) {
    return {p, stride, n->width * float_size(n->type), n_tokens};
}

// Waves of a row, 8 values a thread: 2,560 columns fill five of them and would leave three of eight idle (19.0 us against 15.2 for
// 4,001 tokens in bf16).  Other widths between two counts leave up to half of the waves idle: no forms of their own so far
template <typename F>
static void norm_waves(int width, F go) {
    if (width <= 512) go(std::integral_constant<int, 1>{});
    else if (width <= 1024) go(std::integral_constant<int, 2>{});
    else if (width <= 2048) go(std::integral_constant<int, 4>{});
    else if (width <= 2560) go(std::integral_constant<int, 5>{});
    else if (width <= 4096) go(std::integral_constant<int, 8>{});
    else go(std::integral_constant<int, 16>{});
}
template <typename X>
static void launch_block_norm(const NormArgs& a, hipStream_t st) {
    norm_waves(a.width, [&](auto w) {
        constexpr int W = decltype(w)::value, kRows = norm_threads(W) / (64 * W);
        // a launch takes fewer than 2^32 threads along x, and 2^24 tokens of a workgroup each may be more
        constexpr unsigned kMost = 1u << 20;
        const unsigned groups = (unsigned)((a.n_tokens + kRows - 1) / kRows);
        hipLaunchKernelGGL((k_block_norm<X, 8, W>), dim3(std::min(groups, kMost), (groups + kMost - 1) / kMost), dim3(norm_threads(W)), 0, st, a);
    });
}
template <typename X>
static void launch_block_norm_back(const NormArgs& a, int parts, hipStream_t st) {
    norm_waves(a.width, [&](auto w) {
        constexpr int W = decltype(w)::value, kRows = norm_threads(W) / (64 * W);
        hipLaunchKernelGGL((k_block_norm_back<X, 8, W>), dim3((unsigned)((parts + kRows - 1) / kRows)), dim3(norm_threads(W)), 0, st, a);
    });
}

SABAH_API int sabah_block_norm(const sabah_norm_desc* norm, const void* d_x, size_t x_stride, const void* d_y,
                               size_t y_stride, const float* d_gate, int n_tokens, void* d_out, size_t out_stride,
                               void* d_h, size_t h_stride, void* stream) {
    if (check_norm("block norm", norm, n_tokens)) return -1;
    if (n_tokens && (!d_x || (d_y && !d_out) || (norm->w_before && !d_h))) return fail("block norm: null pointer");
    if (n_tokens && !d_y && !norm->w_before) return fail("block norm: neither y nor a norm before the next block");
    if (n_tokens && !d_y && (d_gate || norm->w_after)) return fail("block norm: a gate or a norm after the block needs y");
    if (!norm_rows_ok(norm, n_tokens, d_x, x_stride) || !norm_rows_ok(norm, n_tokens, d_y, y_stride) ||
        !norm_rows_ok(norm, n_tokens, d_out, out_stride) || !norm_rows_ok(norm, n_tokens, d_h, h_stride))
        return fail("block norm: a stride below a row of %d values, or no multiple of one", norm->width);
    const MemRows x = norm_mem(norm, n_tokens, d_x, x_stride), y = norm_mem(norm, n_tokens, d_y, y_stride);
    const MemRows out = norm_mem(norm, n_tokens, d_y ? d_out : nullptr, out_stride);
    const MemRows h = norm_mem(norm, n_tokens, norm->w_before ? d_h : nullptr, h_stride);
    if (rows_meet(h, x) || rows_meet(h, y) || rows_meet(h, out)) return fail("block norm: h would overwrite x, y or out");
    const bool in_place = d_out == d_x && (n_tokens <= 1 || out_stride == x_stride);
    if (rows_meet(out, y) || (!in_place && rows_meet(out, x))) return fail("block norm: out would overwrite y, or rows of x other than its own");
    if (g_device < 0) return fail("sabah_rt_init has not been called");
    if (!check_sticky()) return -1;
    if (n_tokens == 0) return 0;
    OnDevice dev;
    if (!dev.ok) return -1;
    NormArgs a{};
    a.x = static_cast<const uint8_t*>(d_x);
    a.y = static_cast<const uint8_t*>(d_y);
    a.out = static_cast<uint8_t*>(d_out);
    a.h = static_cast<uint8_t*>(d_h);
    a.x_st = x_stride;
    a.y_st = y_stride;
    a.out_st = out_stride;
    a.h_st = h_stride;
    a.gate = d_gate;
    a.w_after = norm->w_after;
    a.w_before = norm->w_before;
    a.scale = norm->scale;
    a.eps = norm->eps;
    a.n_tokens = n_tokens;
    a.width = norm->width;
    hipStream_t st = pick_stream(stream);
    switch (norm->type) {
    case kTypeF32: launch_block_norm<ExpF32>(a, st); break;
    case kTypeF16: launch_block_norm<ExpF16>(a, st); break;
    default: launch_block_norm<ExpBF16>(a, st); break;
    }
    return ck(hipGetLastError(), "block norm launch") ? 0 : -1;
}

SABAH_API size_t sabah_block_norm_workspace(int width, int n_tokens) {
    const sabah_norm_desc n{nullptr, nullptr, kTypeF32, width, 0.0f, 1.0f};
    if (check_norm("block norm", &n, n_tokens)) return 0;
    int parts, per_part;
    norm_plan(n_tokens, parts, per_part);
    return 2 * align256((size_t)std::max(1, parts) * width * 4);
}

SABAH_API int sabah_block_norm_backward(const sabah_norm_desc* norm, const void* d_out, size_t out_stride, const void* d_y,
                                        size_t y_stride, const float* d_gate, int n_tokens, const void* d_dout,
                                        size_t dout_stride, const void* d_dh, size_t dh_stride, void* d_dx, size_t dx_stride,
                                        void* d_dy, size_t dy_stride, float* d_dgate, float* d_dw_after, float* d_dw_before,
                                        int add_dw, void* d_workspace, size_t workspace_bytes, void* stream) {
    if (check_norm("block norm backward", norm, n_tokens)) return -1;
    const bool after = d_dy != nullptr || !n_tokens, before = norm->w_before != nullptr;
    if (!after && !before) return fail("block norm backward: neither dy nor a norm before the next block");
    if (!after && (d_gate || norm->w_after)) return fail("block norm backward: a gate or a norm after the block needs dy");
    if (n_tokens && ((before && (!d_out || !d_dh || !d_dx)) || (!before && !d_dout) ||
                     (after && !d_y && (norm->w_after || d_gate)) || (d_gate && !d_dgate)))
        return fail("block norm backward: null pointer");
    if ((norm->w_after && !d_dw_after) || (before && !d_dw_before)) return fail("block norm backward: null pointer");
    if (!norm_rows_ok(norm, n_tokens, d_out, out_stride) || !norm_rows_ok(norm, n_tokens, d_y, y_stride) ||
        !norm_rows_ok(norm, n_tokens, d_dout, dout_stride) || !norm_rows_ok(norm, n_tokens, d_dh, dh_stride) ||
        !norm_rows_ok(norm, n_tokens, d_dx, dx_stride) || !norm_rows_ok(norm, n_tokens, d_dy, dy_stride))
        return fail("block norm backward: a stride below a row of %d values, or no multiple of one", norm->width);
    const MemRows out = norm_mem(norm, n_tokens, d_out, out_stride), y = norm_mem(norm, n_tokens, d_y, y_stride);
    const MemRows dout = norm_mem(norm, n_tokens, d_dout, dout_stride), dh = norm_mem(norm, n_tokens, before ? d_dh : nullptr, dh_stride);
    const MemRows dx = norm_mem(norm, n_tokens, before ? d_dx : nullptr, dx_stride), dy = norm_mem(norm, n_tokens, d_dy, dy_stride);
    if (rows_meet(dx, out) || rows_meet(dx, y) || rows_meet(dx, dh) || rows_meet(dy, out) || rows_meet(dy, y) || rows_meet(dy, dh) ||
        rows_meet(dy, dout) || rows_meet(dy, dx))
        return fail("block norm backward: dx or dy would overwrite an input, or each other");
    if (!(d_dx == d_dout && (n_tokens <= 1 || dx_stride == dout_stride)) && rows_meet(dx, dout))
        return fail("block norm backward: dx in place of dout needs its stride and its rows");
    const size_t dw_bytes = norm->width * sizeof(float);
    if (norm->w_after && before && rows_meet({d_dw_after, 0, dw_bytes, 1}, {d_dw_before, 0, dw_bytes, 1}))
        return fail("block norm backward: dw_after and dw_before would overwrite each other");
    int parts, per_part;
    norm_plan(n_tokens, parts, per_part);
    const size_t part = align256((size_t)std::max(1, parts) * norm->width * 4);
    if (!d_workspace || workspace_bytes < 2 * part || (uintptr_t)d_workspace % 16)
        return fail("block norm backward: the workspace must be 16-byte aligned and hold %zu bytes (got %zu)", 2 * part, workspace_bytes);
    if (g_device < 0) return fail("sabah_rt_init has not been called");
    if (!check_sticky()) return -1;
    OnDevice dev;
    if (!dev.ok) return -1;
    NormArgs a{};
    a.x = static_cast<const uint8_t*>(d_out);
    a.y = static_cast<const uint8_t*>(d_y);
    a.dout = static_cast<const uint8_t*>(d_dout);
    a.dh = static_cast<const uint8_t*>(d_dh);
    a.dx = static_cast<uint8_t*>(d_dx);
    a.dy = static_cast<uint8_t*>(d_dy);
    a.x_st = out_stride;
    a.y_st = y_stride;
    a.dout_st = dout_stride;
    a.dh_st = dh_stride;
    a.dx_st = dx_stride;
    a.dy_st = dy_stride;
    a.gate = d_gate;
    a.dgate = d_dgate;
    a.w_after = norm->w_after;
    a.w_before = norm->w_before;
    a.part_after = static_cast<float*>(d_workspace);
    a.part_before = reinterpret_cast<float*>(static_cast<uint8_t*>(d_workspace) + part);
    a.scale = norm->scale;
    a.eps = norm->eps;
    a.n_tokens = n_tokens;
    a.width = norm->width;
    a.per_part = per_part;
    hipStream_t st = pick_stream(stream);
    if (n_tokens) {
        switch (norm->type) {
        case kTypeF32: launch_block_norm_back<ExpF32>(a, parts, st); break;
        case kTypeF16: launch_block_norm_back<ExpF16>(a, parts, st); break;
        default: launch_block_norm_back<ExpBF16>(a, parts, st); break;
        }
        if (!ck(hipGetLastError(), "block norm backward launch")) return -1;
    } else if (add_dw) {
        return 0;
    }
    NormSumArgs s{};
    int sums = 0;
    if (norm->w_after) {
        s.part[sums] = a.part_after;
        s.out[sums++] = d_dw_after;
    }
    if (before) {
        s.part[sums] = a.part_before;
        s.out[sums++] = d_dw_before;
    }
    if (!sums) return 0;
    s.parts = parts;
    s.width = norm->width;
    s.add = add_dw != 0;
    hipLaunchKernelGGL(k_block_norm_sum, dim3((unsigned)((norm->width + kNormSumCols - 1) / kNormSumCols), (unsigned)sums), dim3(1024), 0, st, s);
    return ck(hipGetLastError(), "block norm sum launch") ? 0 : -1;
}

// ---------------------------------------------------------------------------
// experts
// ---------------------------------------------------------------------------
static int check_groups(const char* what, int n_ids, int n_tokens, int n_experts) {
    if (n_ids <= 0 || n_tokens < 0 || (long long)n_ids * n_tokens > 1 << 24)
        return fail("%s: n_ids=%d, n_tokens=%d give no rows, or too many", what, n_ids, n_tokens);
    if (n_experts <= 0 || n_experts > kExpMaxExperts) return fail("%s: n_experts %d outside [1, %d]", what, n_experts, kExpMaxExperts);
    return 0;
}
static int check_groups_buffer(const char* what, const ExpertPlan& p, const void* d_groups, size_t bytes) {
    if (!d_groups || bytes < p.words * 4 || (uintptr_t)d_groups % 16)
        return fail("%s: the groups must be 16-byte aligned and hold %zu bytes (got %zu)", what, p.words * 4, bytes);
    return 0;
}

// rows [n_tokens][n_ids] of `bytes`, the longer stride outside; own: whether the rows are apart from each other
static MemRows expert_mem(const void* p, size_t id, size_t tok, int n_ids, int n_tokens, size_t bytes, bool* own = nullptr) {
    if (n_ids == 1) id = 0;
    if (n_tokens <= 1) tok = 0;
    const bool tokens = tok >= id;
    const size_t outer = tokens ? tok : id, inner = tokens ? id : tok;
    const int n = tokens ? n_tokens : n_ids, m = tokens ? n_ids : n_tokens;
    const MemRows r{p, outer, (size_t)(m - 1) * inner + bytes, n_tokens ? n : 0, inner, bytes, m};
    if (own) *own = (m <= 1 || inner >= bytes) && (n <= 1 || outer >= r.bytes);
    return r;
}
// the groups' memory: kernels take rows' numbers and tiles from it, so nothing else may be written there
static MemRows groups_mem(const ExpertPlan& p, const void* d_groups) { return {d_groups, 0, p.words * 4, 1}; }

SABAH_API size_t sabah_expert_groups_bytes(int n_ids, int n_tokens, int n_experts) {
    if (check_groups("expert groups", n_ids, n_tokens, n_experts)) return 0;
    return expert_plan(n_ids, n_tokens, n_experts).words * 4;
}

SABAH_API int sabah_expert_group(const int32_t* d_ids, size_t ids_id_stride, size_t ids_token_stride, int n_ids, int n_tokens,
                                 int n_experts, void* d_groups, size_t groups_bytes, void* stream) {
    if (check_groups("expert groups", n_ids, n_tokens, n_experts)) return -1;
    if (n_tokens && !d_ids) return fail("expert groups: null pointer");
    if (!stride_ok(ids_id_stride) || !stride_ok(ids_token_stride)) return fail("expert groups: strides are in bytes and multiples of 4");
    ExpertGroupArgs a{};
    a.p = expert_plan(n_ids, n_tokens, n_experts);
    if (check_groups_buffer("expert groups", a.p, d_groups, groups_bytes)) return -1;
    if (rows_meet(groups_mem(a.p, d_groups), expert_mem(d_ids, ids_id_stride, ids_token_stride, n_ids, n_tokens, 4)))
        return fail("expert groups: the groups would overwrite the ids");
    if (g_device < 0) return fail("sabah_rt_init has not been called");
    if (!check_sticky()) return -1;
    OnDevice dev;
    if (!dev.ok) return -1;
    a.ids = reinterpret_cast<const uint8_t*>(d_ids);
    a.ids_id = ids_id_stride;
    a.ids_tok = ids_token_stride;
    a.g = static_cast<uint32_t*>(d_groups);
    a.err = g_err_dev;
    hipStream_t st = pick_stream(stream);
    const int keys = n_experts + 2;
    constexpr auto lds_of = [](int keys, bool sums) { return kExpGroupWaves * (8 + (keys + 1) / 2 * 4) + (sums ? 2 : 1) * keys * 4; };
    static_assert(lds_of(kExpMaxExperts + 2, false) <= 160 * 1024, "a workgroup's LDS");   // with sums 4,096 experts have more: below
    const dim3 grid((unsigned)a.p.chunks), block(kExpGroupThreads);
    if (a.p.n_rows <= kExpFewGroup) {
        hipLaunchKernelGGL(k_expert_group_few, dim3(1), dim3(256), 0, st, a);
    } else if (a.p.chunks == 1) {
        const int lds = lds_of(keys, false);
        if (!ck(fit_lds(k_expert_place<kPlaceAlone>, lds, lds), "expert groups LDS")) return -1;
        hipLaunchKernelGGL(k_expert_place<kPlaceAlone>, grid, block, (uint32_t)lds, st, a);
    } else {
        hipLaunchKernelGGL(k_expert_count, grid, block, (uint32_t)keys * 4, st, a);
        const bool sums = a.p.chunks <= kExpSumChunks && lds_of(keys, true) <= g_max_lds;
        const int lds = lds_of(keys, sums);
        if (sums) {
            if (!ck(fit_lds(k_expert_place<kPlaceSum>, lds, lds), "expert groups LDS")) return -1;
            hipLaunchKernelGGL(k_expert_place<kPlaceSum>, grid, block, (uint32_t)lds, st, a);
        } else {
            hipLaunchKernelGGL(k_expert_scan, dim3(1), block, (uint32_t)keys * 4, st, a);
            if (!ck(fit_lds(k_expert_place<kPlaceScanned>, lds, lds), "expert groups LDS")) return -1;
            hipLaunchKernelGGL(k_expert_place<kPlaceScanned>, grid, block, (uint32_t)lds, st, a);
        }
    }
    return ck(hipGetLastError(), "expert groups launch") ? 0 : -1;
}

static int check_experts(const char* what, const sabah_expert_desc* E, const void* d_x, size_t x_id_stride, int x_rows,
                         size_t x_token_stride, int n_ids, int n_tokens) {
    if (!E || !E->w) return fail("%s: null experts", what);
    if (!float_type(E->type)) return fail("%s: type %d is none of F32 (0), F16 (1), BF16 (30)", what, E->type);
    if (check_groups(what, n_ids, n_tokens, E->n_experts)) return -1;
    if (E->k <= 0 || E->rows <= 0 || E->k > 1 << 20 || E->rows > 1 << 20)
        return fail("%s: invalid geometry (k=%d rows=%d)", what, E->k, E->rows);
    if (n_tokens && !d_x) return fail("%s: null pointer", what);
    if (x_rows != 1 && x_rows != n_ids) return fail("%s: %d input rows, expected 1 or n_ids=%d", what, x_rows, n_ids);
    if (x_id_stride % float_size(E->type) || x_token_stride % float_size(E->type))
        return fail("%s: strides are in bytes and whole values", what);
    return 0;
}
static MemRows expert_weights(const sabah_expert_desc* E, const void* p, size_t value) {
    return {p, 0, (size_t)E->n_experts * E->rows * E->k * value, 1};
}
static ExpertArgs expert_args(const sabah_expert_desc* E, const void* d_x, size_t x_id_stride, int x_rows, size_t x_token_stride,
                              const void* d_groups, int n_ids, int n_tokens) {
    ExpertArgs a{};
    a.g = static_cast<const uint32_t*>(d_groups);
    a.p = expert_plan(n_ids, n_tokens, E->n_experts);
    a.w = static_cast<const uint8_t*>(E->w);
    a.k = E->k;
    a.rows = E->rows;
    a.x = static_cast<const uint8_t*>(d_x);
    a.x_id = x_id_stride;
    a.x_tok = x_token_stride;
    a.x_rows = x_rows;
    a.err = g_err_dev;
    return a;
}
// a launch takes fewer than 2^32 threads along x
static int expert_grid(const char* what, long long works, int threads, dim3& grid) {
    if (works > ((1ll << 32) - 1) / threads - 8) return fail("%s: %lld tiles are too many for one call", what, works);
    grid = dim3((unsigned)((works + 7) / 8 * 8));
    return 0;
}


template <typename X, int MODE>
static int launch_expert_gemm(const char* what, const ExpertArgs& a, hipStream_t st) {
    typedef ExpGemm<X, MODE> G;
    const long long cols = ((MODE == kModeForward ? a.rows : a.k) + G::BN - 1) / G::BN;
    dim3 grid;
    if (expert_grid(what, (MODE == kModeDw ? (long long)a.p.n_experts * ((a.rows + G::BM - 1) / G::BM) : a.p.max_tiles) * cols, kExpThreads, grid)) return -1;
    if (!ck(fit_lds(k_expert_gemm<X, MODE>, G::kLdsAll, G::kLdsAll), what)) return -1;
    hipLaunchKernelGGL((k_expert_gemm<X, MODE>), grid, dim3(kExpThreads), G::kLdsAll, st, a);
    return ck(hipGetLastError(), what) ? 0 : -1;
}
// whether every row of x, dy and out, and of the weights, is whole multiples of 16 bytes from an aligned start
static bool expert_aligned(const ExpertArgs& a, int es) {
    const size_t all = (size_t)(uintptr_t)a.w | (uintptr_t)a.x | (uintptr_t)a.dy | (uintptr_t)a.out | a.x_id | a.x_tok | a.dy_id |
                       a.dy_tok | a.out_id | a.out_tok | (size_t)a.k * es | (size_t)a.rows * es;
    return all % 16 == 0;
}
template <typename X, int MODE, int BM, int BN, int WM, int WN, int KB, int S, int OCC>
static int launch_expert_fast(const char* what, const ExpertArgs& a, hipStream_t st) {
    typedef ExpFast<X, MODE, BM, BN, WM, WN, KB, S> G;
    const long long cols = ((MODE == kModeForward ? a.rows : a.k) + BN - 1) / BN;
    dim3 grid;
    if (expert_grid(what, (BM == kExpLarge ? a.p.max_large : a.p.max_tiles) * cols, 64 * G::NW, grid)) return -1;
    auto kernel = k_expert_fast<X, MODE, BM, BN, WM, WN, KB, S, OCC>;
    if (!ck(fit_lds(kernel, G::kLds, G::kLds), what)) return -1;
    hipLaunchKernelGGL(kernel, grid, dim3(64 * G::NW), G::kLds, st, a);
    return ck(hipGetLastError(), what) ? 0 : -1;
}
template <typename X, int BM, int BN, int WM, int WN, int KB, int S, int OCC>
static int launch_expert_dw(const char* what, const ExpertArgs& a, hipStream_t st) {
    typedef ExpFast<X, kModeDw, BM, BN, WM, WN, KB, S> G;
    dim3 grid;
    if (expert_grid(what, (long long)a.p.n_experts * ((a.rows + BM - 1) / BM) * ((a.k + BN - 1) / BN), 64 * G::NW, grid)) return -1;
    auto kernel = k_expert_dw<X, BM, BN, WM, WN, KB, S, OCC>;
    if (!ck(fit_lds(kernel, G::kLds, G::kLds), what)) return -1;
    hipLaunchKernelGGL(kernel, grid, dim3(64 * G::NW), G::kLds, st, a);
    return ck(hipGetLastError(), what) ? 0 : -1;
}
// Which tile, of 16-bit types (us in bf16, 8 experts unless said, 2,048 -> 768; rows to an expert):
//   128 x 64   while tiles of 128 x 256 are too few for the card: forward at 256 rows 20.4 against 32.5, at 512 30.2 and 33.8,
//              at 1,024 (216 tiles) 48.7 and 36.8; dx at 128 rows 13.8 and 18.8, at 512 (288 tiles) 40.7 and 26.8
//   256 x 256  forward, from 384 rows and three quarters of the card's tiles: of 128 experts at 256 rows 186 against 168, at 384
//              208 and 225, at 512 259 and 279; at 8,192 rows 210 and 240, at 2,048 58 and 67, at 1,024 (96 tiles) 54 and 37.  Of
//              dx, whose sums are shorter, 353 and 330 (128 experts, 512 rows)
//   128 x 256  else, and for dW: 338 against 356 with 256 x 256, 346 with 128 x 128 (128 experts, 256 rows, 768 -> 2,048); few tiles
//              are not faster in 128 x 64 (14.4, 15.4)
// f32's products take 64 cycles where loads take few: 128 x 128 with all four waves on all rows, so that a last tile's missing rows
// are missing from each (600 rows of 8 experts: dx 53 us; dW in 128 x 64 46 - 52, in 128 x 128 50 - 58).
constexpr int kExpLargeRows = 384;
template <typename X, int MODE>
static int launch_expert_product(const char* what, const ExpertArgs& a, hipStream_t st) {
    if (!expert_aligned(a, (int)sizeof(typename X::S))) return launch_expert_gemm<X, MODE>(what, a, st);
    const int R = a.p.n_rows, E = a.p.n_experts, cols = ((MODE == kModeForward ? a.rows : a.k) + 255) / 256;
    if constexpr (sizeof(typename X::S) == 4) {
        if constexpr (MODE == kModeDw) return launch_expert_dw<X, 128, 64, 2, 2, 64, 2, 4>(what, a, st);
        else return launch_expert_fast<X, MODE, 128, 128, 1, 4, 64, 4, 2>(what, a, st);
    } else if constexpr (MODE == kModeDw) {
        return launch_expert_dw<X, 128, 256, 2, 4, 64, 3, 4>(what, a, st);
    } else {
        if ((long long)(R / kExpTile + std::min(R, E)) * cols < g_num_cu * 7 / 10)
            return launch_expert_fast<X, MODE, 128, 64, 2, 2, 64, 4, 3>(what, a, st);
        if (MODE == kModeForward && R / kExpLargeRows >= E && (long long)(R / kExpLarge) * cols >= g_num_cu * 3 / 4)
            return launch_expert_fast<X, MODE, 256, 256, 2, 4, 64, 3, 2>(what, a, st);
        return launch_expert_fast<X, MODE, 128, 256, 2, 4, 64, 3, 4>(what, a, st);
    }
}
template <typename X, int NW>
static int launch_expert_rows(const ExpertArgs& a, hipStream_t st) {
    constexpr int NT = 2;
    dim3 grid;
    if (expert_grid("expert product", (long long)a.p.max_small * ((a.rows + 16 * NT - 1) / (16 * NT)), 64 * NW, grid)) return -1;
    hipLaunchKernelGGL((k_expert_rows<X, NT, NW>), grid, dim3(64 * NW), 0, st, a);
    return ck(hipGetLastError(), "expert product launch") ? 0 : -1;
}
template <typename X>
static int launch_expert_mul(const ExpertArgs& a, hipStream_t st) {
    if ((long long)a.p.n_rows > (long long)kExpFewRows * a.p.n_experts)
        return launch_expert_product<X, kModeForward>("expert product launch", a, st);
    return (size_t)a.k * sizeof(typename X::S) >= 2048 ? launch_expert_rows<X, 8>(a, st) : launch_expert_rows<X, 4>(a, st);
}

SABAH_API int sabah_expert_mul(const sabah_expert_desc* experts, const void* d_x, size_t x_id_stride, int x_rows,
                               size_t x_token_stride, const void* d_groups, size_t groups_bytes, int n_ids, int n_tokens,
                               void* d_y, size_t y_id_stride, size_t y_token_stride, void* stream) {
    if (check_experts("expert product", experts, d_x, x_id_stride, x_rows, x_token_stride, n_ids, n_tokens)) return -1;
    if (n_tokens && !d_y) return fail("expert product: null pointer");
    if (y_id_stride % float_size(experts->type) || y_token_stride % float_size(experts->type))
        return fail("expert product: strides are in bytes and whole values");
    const size_t es = float_size(experts->type);
    bool own;
    const MemRows x = expert_mem(d_x, x_id_stride, x_token_stride, x_rows, n_tokens, experts->k * es);
    const MemRows y = expert_mem(d_y, y_id_stride, y_token_stride, n_ids, n_tokens, experts->rows * es, &own);
    if (n_tokens && !own) return fail("expert product: rows of y overlap");
    if (rows_meet(y, x) || rows_meet(y, expert_weights(experts, experts->w, es))) return fail("expert product: y would overwrite x or the weights");
    ExpertArgs a = expert_args(experts, d_x, x_id_stride, x_rows, x_token_stride, d_groups, n_ids, n_tokens);
    if (check_groups_buffer("expert product", a.p, d_groups, groups_bytes)) return -1;
    if (rows_meet(y, groups_mem(a.p, d_groups))) return fail("expert product: y would overwrite the groups");
    if (g_device < 0) return fail("sabah_rt_init has not been called");
    if (!check_sticky()) return -1;
    if (n_tokens == 0) return 0;
    OnDevice dev;
    if (!dev.ok) return -1;
    a.out = static_cast<uint8_t*>(d_y);
    a.out_id = y_id_stride;
    a.out_tok = y_token_stride;
    hipStream_t st = pick_stream(stream);
    switch (experts->type) {
    case kTypeF32: return launch_expert_mul<ExpF32>(a, st);
    case kTypeF16: return launch_expert_mul<ExpF16>(a, st);
    default: return launch_expert_mul<ExpBF16>(a, st);
    }
}

template <typename X>
static int launch_expert_back(const ExpertArgs& a, hipStream_t st) {
    if (a.out && a.p.n_rows && launch_expert_product<X, kModeDx>("expert product's gradient launch", a, st)) return -1;
    return a.dw ? launch_expert_product<X, kModeDw>("expert weights' gradient launch", a, st) : 0;
}

SABAH_API int sabah_expert_mul_backward(const sabah_expert_desc* experts, const void* d_x, size_t x_id_stride, int x_rows,
                                        size_t x_token_stride, const void* d_groups, size_t groups_bytes, int n_ids,
                                        int n_tokens, const void* d_dy, size_t dy_id_stride, size_t dy_token_stride,
                                        void* d_dx, size_t dx_id_stride, size_t dx_token_stride, float* d_dw, int add_dw,
                                        void* stream) {
    if (check_experts("expert product backward", experts, d_x, x_id_stride, x_rows, x_token_stride, n_ids, n_tokens)) return -1;
    if (n_tokens && !d_dy) return fail("expert product backward: null pointer");
    const size_t es = float_size(experts->type);
    if (dy_id_stride % es || dy_token_stride % es || dx_id_stride % es || dx_token_stride % es)
        return fail("expert product backward: strides are in bytes and whole values");
    bool own;
    const MemRows x = expert_mem(d_x, x_id_stride, x_token_stride, x_rows, n_tokens, experts->k * es);
    const MemRows dy = expert_mem(d_dy, dy_id_stride, dy_token_stride, n_ids, n_tokens, experts->rows * es);
    const MemRows dx = expert_mem(d_dx, dx_id_stride, dx_token_stride, n_ids, n_tokens, experts->k * es, &own);
    const MemRows w = expert_weights(experts, experts->w, es), dw = expert_weights(experts, d_dw, sizeof(float));
    if (n_tokens && d_dx && !own) return fail("expert product backward: rows of dx overlap");
    if (rows_meet(dx, x) || rows_meet(dx, dy) || rows_meet(dx, w)) return fail("expert product backward: dx would overwrite x, dy or the weights");
    if (rows_meet(dw, x) || rows_meet(dw, dy) || rows_meet(dw, w) || rows_meet(dw, dx))
        return fail("expert product backward: dw would overwrite x, dy, dx or the weights");
    ExpertArgs a = expert_args(experts, d_x, x_id_stride, x_rows, x_token_stride, d_groups, n_ids, n_tokens);
    if (check_groups_buffer("expert product backward", a.p, d_groups, groups_bytes)) return -1;
    if (rows_meet(dx, groups_mem(a.p, d_groups)) || rows_meet(dw, groups_mem(a.p, d_groups)))
        return fail("expert product backward: dx or dw would overwrite the groups");
    if (g_device < 0) return fail("sabah_rt_init has not been called");
    if (!check_sticky()) return -1;
    OnDevice dev;
    if (!dev.ok) return -1;
    a.dy = static_cast<const uint8_t*>(d_dy);
    a.dy_id = dy_id_stride;
    a.dy_tok = dy_token_stride;
    a.out = static_cast<uint8_t*>(d_dx);
    a.out_id = dx_id_stride;
    a.out_tok = dx_token_stride;
    a.dw = d_dw;
    a.add = add_dw != 0;
    hipStream_t st = pick_stream(stream);
    switch (experts->type) {
    case kTypeF32: return launch_expert_back<ExpF32>(a, st);
    case kTypeF16: return launch_expert_back<ExpF16>(a, st);
    default: return launch_expert_back<ExpBF16>(a, st);
    }
}

// ---------------------------------------------------------------------------
// AdamW
// ---------------------------------------------------------------------------
static int check_adamw_tensors(const sabah_adamw_tensor* t, int n, long long& chunks, long long& values) {
    if (n <= 0 || n > 1 << 20 || !t) return fail("adamw: %d tensors, expected 1 to %d", n, 1 << 20);
    struct Range {
        uintptr_t lo, hi;
        bool written;
    };
    std::vector<Range> all;
    chunks = values = 0;
    for (int i = 0; i < n; ++i) {
        if (!float_type(t[i].p_type) || !float_type(t[i].g_type)) return fail("adamw: tensor %d has types %d and %d, each F32 (0), F16 (1) or BF16 (30)", i, t[i].p_type, t[i].g_type);
        if (t[i].n < 0 || t[i].n > 1ll << 40) return fail("adamw: tensor %d of %lld values", i, t[i].n);
        if (t[i].n && (!t[i].p || !t[i].g)) return fail("adamw: tensor %d is null", i);
        if (t[i].master && t[i].p_type == kTypeF32) return fail("adamw: tensor %d is f32 and has a master copy", i);
        if (!(t[i].decay >= 0.0 && t[i].decay < __builtin_inf())) return fail("adamw: tensor %d has decay %g", i, t[i].decay);
        chunks += (t[i].n + kAdamChunk - 1) / kAdamChunk;
        values += (t[i].n + kAdamBlock - 1) / kAdamBlock * kAdamBlock;
        const uintptr_t p = (uintptr_t)t[i].p, g = (uintptr_t)t[i].g, m = (uintptr_t)t[i].master;
        if (!t[i].n) continue;
        if (p % float_size(t[i].p_type) || g % float_size(t[i].g_type) || m % 4) return fail("adamw: tensor %d is not aligned to its values", i);
        all.push_back({p, p + t[i].n * float_size(t[i].p_type), true});
        all.push_back({g, g + t[i].n * float_size(t[i].g_type), false});
        if (m) all.push_back({m, m + t[i].n * 4, true});
    }
    if (chunks >= 1 << 24) return fail("adamw: %lld values are too many for one step", values);
    std::sort(all.begin(), all.end(), [](const Range& x, const Range& y) { return x.lo < y.lo; });
    uintptr_t any = 0, written = 0;
    for (const Range& r : all) {
        if (r.lo < written || (r.written && r.lo < any)) return fail("adamw: a weight shares memory with another tensor");
        any = std::max(any, r.hi);
        if (r.written) written = std::max(written, r.hi);
    }
    return 0;
}
static size_t adamw_chunks_at(int n) { return align256((size_t)n * sizeof(AdamTensor)); }

// the check keeps a list of the tensors' memory: without memory for it the call fails, as any other
static int check_adamw_table(const sabah_adamw_tensor* t, int n, long long& chunks, long long& values) {
    try {
        return check_adamw_tensors(t, n, chunks, values);
    } catch (const std::exception& e) {
        return fail("adamw: %s", e.what());
    }
}

SABAH_API size_t sabah_adamw_table_bytes(const sabah_adamw_tensor* tensors, int n_tensors, long long* n_values) {
    long long chunks, values;
    if (!n_values) {
        fail("adamw: null pointer");
        return 0;
    }
    if (check_adamw_table(tensors, n_tensors, chunks, values)) return 0;
    *n_values = values;
    return adamw_chunks_at(n_tensors) + (size_t)chunks * sizeof(AdamChunk);
}

SABAH_API int sabah_adamw_table(const sabah_adamw_tensor* tensors, int n_tensors, void* table, size_t table_bytes) {
    long long chunks, values;
    if (check_adamw_table(tensors, n_tensors, chunks, values)) return -1;
    const size_t need = adamw_chunks_at(n_tensors) + (size_t)chunks * sizeof(AdamChunk);
    if (!table || table_bytes != need) return fail("adamw: the table has %zu bytes (got %zu)", need, table_bytes);
    std::memset(table, 0, need);
    AdamTensor* t = static_cast<AdamTensor*>(table);
    AdamChunk* c = reinterpret_cast<AdamChunk*>(static_cast<uint8_t*>(table) + adamw_chunks_at(n_tensors));
    long long at = 0;
    for (int i = 0; i < n_tensors; ++i) {
        const sabah_adamw_tensor& s = tensors[i];
        t[i] = AdamTensor{static_cast<uint8_t*>(s.p), static_cast<const uint8_t*>(s.g), s.master, s.decay, s.n, at, s.p_type, s.g_type};
        for (long long k = 0; k * kAdamChunk < s.n; ++k) *c++ = AdamChunk{i, (int)k};
        at += (s.n + kAdamBlock - 1) / kAdamBlock * kAdamBlock;
    }
    return 0;
}

SABAH_API size_t sabah_adamw_workspace(void) { return align256(kAdamNormGroups * sizeof(double)) + align256(sizeof(AdamScalars)); }

SABAH_API int sabah_adamw_step(const sabah_adamw_desc* o, void* stream) {
    if (!o || !o->table || !o->step) return fail("adamw: null pointer");
    const bool unbiased = o->bits == (8 | SABAH_ADAMW_UNBIASED);
    const int bits = unbiased ? 8 : o->bits;
    if (bits != 32 && bits != 8) return fail("adamw: moments of %d bits, expected 32 or 8", o->bits);
    if ((uintptr_t)o->m % 16 || (uintptr_t)o->v % 16 || (uintptr_t)o->table % 16) return fail("adamw: the table and the moments must be 16-byte aligned");
    if (!(o->beta1 >= 0.0 && o->beta1 < 1.0 && o->beta2 >= 0.0 && o->beta2 < 1.0)) return fail("adamw: betas %g, %g outside [0, 1)", o->beta1, o->beta2);
    // the step adds it in f32: what vanishes there would divide 0 by 0
    if (!(o->eps >= 1.2e-38 && o->eps < 3.4e38)) return fail("adamw: eps %g outside f32's positive numbers", o->eps);
    if (!(o->lr >= 0.0 && o->lr < __builtin_inf())) return fail("adamw: lr must be finite and not negative");
    if (!(o->grad_scale > 0.0 && o->grad_scale < __builtin_inf())) return fail("adamw: grad_scale must be positive and finite");
    if (o->norm && !(o->max_norm > 0.0)) return fail("adamw: max_norm must be positive");
    const size_t at = o->n_tensors > 0 ? adamw_chunks_at(o->n_tensors) : 0;
    if (o->n_tensors <= 0 || o->table_bytes < at || (o->table_bytes - at) % sizeof(AdamChunk) || (o->table_bytes - at) / sizeof(AdamChunk) >= 1u << 24)
        return fail("adamw: %zu bytes are no table of %d tensors", o->table_bytes, o->n_tensors);
    if (o->table_bytes > at && (!o->m || !o->v || (bits == 8 && (!o->m_scale || !o->v_scale)))) return fail("adamw: null pointer");
    const size_t ws = sabah_adamw_workspace();
    if (!o->workspace || o->workspace_bytes < ws || (uintptr_t)o->workspace % 16)
        return fail("adamw: the workspace must be 16-byte aligned and hold %zu bytes (got %zu)", ws, o->workspace_bytes);
    if (g_device < 0) return fail("sabah_rt_init has not been called");
    if (!check_sticky()) return -1;
    OnDevice dev;
    if (!dev.ok) return -1;
    AdamArgs a{};
    a.tensors = static_cast<const AdamTensor*>(o->table);
    a.chunks = reinterpret_cast<const AdamChunk*>(static_cast<const uint8_t*>(o->table) + at);
    a.n_chunks = (int)((o->table_bytes - at) / sizeof(AdamChunk));
    a.bits = bits;
    a.m = o->m;
    a.v = o->v;
    a.m_scale = o->m_scale;
    a.v_scale = o->v_scale;
    a.b1 = o->beta1;
    a.b2 = o->beta2;
    a.eps = o->eps;
    a.lr = o->lr;
    a.lr_dev = o->d_lr;
    a.grad_scale = o->grad_scale;
    a.max_norm = o->max_norm;
    a.step = o->step;
    a.norm = o->norm;
    a.part = static_cast<double*>(o->workspace);
    a.s = reinterpret_cast<AdamScalars*>(static_cast<uint8_t*>(o->workspace) + align256(kAdamNormGroups * sizeof(double)));
    a.parts = std::min(kAdamNormGroups, a.n_chunks);
    hipStream_t st = pick_stream(stream);
    if (a.norm && a.parts) hipLaunchKernelGGL(k_adamw_norm, dim3((unsigned)a.parts), dim3(kAdamThreads), 0, st, a);
    hipLaunchKernelGGL(k_adamw_begin, dim3(1), dim3(a.norm ? 1024 : 64), 0, st, a);
    if (a.n_chunks) {
        const dim3 grid((unsigned)a.n_chunks), block(kAdamThreads);
        if (bits == 32) hipLaunchKernelGGL((k_adamw_step<32, false>), grid, block, 0, st, a);
        else if (!unbiased) hipLaunchKernelGGL((k_adamw_step<8, false>), grid, block, 0, st, a);
        else hipLaunchKernelGGL((k_adamw_step<8, true>), grid, block, 0, st, a);
    }
    return ck(hipGetLastError(), "adamw launch") ? 0 : -1;
}

static int adamw_moments(bool encode, void* m_code, void* v_code, float* m_scale, float* v_scale, long long n_values, float* m,
                         float* v, void* stream) {
    if (n_values < 0 || n_values % kAdamBlock || n_values >= 1ll << 35) return fail("adamw: %lld values are no whole blocks of %d", n_values, kAdamBlock);
    if (n_values && (!m_code || !v_code || !m_scale || !v_scale || !m || !v)) return fail("adamw: null pointer");
    if (((uintptr_t)m_code | (uintptr_t)v_code | (uintptr_t)m | (uintptr_t)v) % 16) return fail("adamw: moments must be 16-byte aligned");
    if (g_device < 0) return fail("sabah_rt_init has not been called");
    if (!check_sticky()) return -1;
    if (!n_values) return 0;
    OnDevice dev;
    if (!dev.ok) return -1;
    const AdamMomentArgs a{static_cast<uint8_t*>(m_code), static_cast<uint8_t*>(v_code), m_scale, v_scale, m, v, n_values / kAdamBlock};
    constexpr long long kMost = 1 << 20;                   // fewer than 2^32 threads along x
    const long long groups = (a.blocks + 3) / 4;
    const dim3 grid((unsigned)std::min(groups, kMost), (unsigned)((groups + kMost - 1) / kMost));
    if (encode) hipLaunchKernelGGL(k_adamw_encode, grid, dim3(kAdamThreads), 0, pick_stream(stream), a);
    else hipLaunchKernelGGL(k_adamw_decode, grid, dim3(kAdamThreads), 0, pick_stream(stream), a);
    return ck(hipGetLastError(), "adamw moments launch") ? 0 : -1;
}
SABAH_API int sabah_adamw_moments_read(const void* m_code, const void* v_code, const float* m_scale, const float* v_scale,
                                       long long n_values, float* m, float* v, void* stream) {
    return adamw_moments(false, const_cast<void*>(m_code), const_cast<void*>(v_code), const_cast<float*>(m_scale),
                         const_cast<float*>(v_scale), n_values, m, v, stream);
}
SABAH_API int sabah_adamw_moments_write(const float* m, const float* v, long long n_values, void* m_code, void* v_code,
                                        float* m_scale, float* v_scale, void* stream) {
    return adamw_moments(true, m_code, v_code, m_scale, v_scale, n_values, const_cast<float*>(m), const_cast<float*>(v), stream);
}
