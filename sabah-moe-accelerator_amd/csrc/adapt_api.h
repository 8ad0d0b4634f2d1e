// C-ABI entry points of the operators that adapt a frozen bank: adapters
// (lora_kernels.h), the router's losses and gradient (balance_kernels.h).
// Included by sabah_rt.hip after its helpers (fail, ck, check_sticky).
// Their device scratch is the caller's: calls on different streams, or captured in
// different graphs, share nothing.
#pragma once

// The calling thread's device is the library's while one lives (a program with
// several GPUs may have another one current).
struct OnDevice {
    int before = -1;
    bool ok = true;
    OnDevice() {
        int now = -1;
        if (!ck(hipGetDevice(&now), "current device")) {
            ok = false;
        } else if (now != g_device) {
            ok = ck(hipSetDevice(g_device), "set device");
            before = now;
        }
    }
    ~OnDevice() {
        if (before >= 0) (void)hipSetDevice(before);
    }
};

constexpr size_t align256(size_t n) { return (n + 255) / 256 * 256; }

// ---------------------------------------------------------------------------
// balance loss, counts; the logits' gradient
// ---------------------------------------------------------------------------
// Workgroups of k_balance_rows to aim at: enough to fill the chip, few enough that adding up their sums stays small
constexpr int kBalanceGroups = 512;

// a group's tokens in runs: multiples of four, one for each wave of a workgroup
static void balance_plan(int n_tokens, int n_groups, int& chunks, int& chunk_len) {
    const int len = n_tokens / n_groups;
    const int most = std::max(1, kBalanceGroups / n_groups);
    chunk_len = std::max(4, ((len + most - 1) / most + 3) / 4 * 4);
    chunks = std::max(1, (len + chunk_len - 1) / chunk_len);
}

struct BalanceSpace {
    size_t p, c, z, loss, group, ticket, bytes;
};
static BalanceSpace balance_space(int n_tokens, int n_experts, int n_groups) {
    int chunks, len;
    balance_plan(n_tokens, n_groups, chunks, len);
    const size_t parts = (size_t)n_groups * chunks;
    BalanceSpace s{};
    s.p = 0;
    s.c = s.p + align256(parts * n_experts * 4);
    s.z = s.c + align256(parts * n_experts * 4);
    s.loss = s.z + align256(parts * 8);
    s.group = s.loss + align256((size_t)n_groups * ((n_experts + kBalanceCols - 1) / kBalanceCols) * 8);
    s.ticket = s.group + align256((size_t)n_groups * 16);
    s.bytes = s.ticket + 256;
    return s;
}

static int check_router_shape(const char* what, int n_tokens, int n_experts, int n_used, int n_groups) {
    if (n_experts <= 0 || n_experts > kRouteThreads * kRouteMaxPerThread)
        return fail("%s: n_experts %d outside [1, %d]", what, n_experts, kRouteThreads * kRouteMaxPerThread);
    if (n_used <= 0 || n_used > n_experts || n_used > kRouteMaxUsed)
        return fail("%s: n_used %d outside [1, min(n_experts, %d)]", what, n_used, kRouteMaxUsed);
    if (n_tokens < 0 || n_tokens > 1 << 24) return fail("%s: n_tokens %d outside [0, %d]", what, n_tokens, 1 << 24);
    if (n_groups <= 0 || n_groups > 65535 || n_tokens % n_groups)
        return fail("%s: n_groups %d does not divide %d tokens, or is outside [1, 65535]", what, n_groups, n_tokens);
    return 0;
}

SABAH_API size_t sabah_moe_balance_workspace(int n_tokens, int n_experts, int n_groups) {
    if (check_router_shape("balance", n_tokens, n_experts, 1, n_groups)) return 0;
    return balance_space(n_tokens, n_experts, n_groups).bytes;
}

template <int PER, int VEC, int W>
static void launch_balance_rows(const BalanceArgs& a, hipStream_t st) {
    hipLaunchKernelGGL((k_balance_rows<PER, VEC, W>), dim3((unsigned)a.chunks, (unsigned)a.n_groups), dim3(row_threads(W)),
                       (uint32_t)a.n_experts * 8, st, a);
}

SABAH_API int sabah_moe_balance(const float* d_logits, size_t logits_stride, const int32_t* d_ids,
                                const uint8_t* d_mask, int n_tokens, int n_experts, int n_used, int n_groups,
                                int32_t* d_counts, float* d_mean_p, float* d_losses, int32_t* d_n_valid,
                                void* d_workspace, size_t workspace_bytes, void* stream) {
    if (check_router_shape("balance", n_tokens, n_experts, n_used, n_groups)) return -1;
    if (((!d_logits || !d_ids) && n_tokens) || !d_counts || !d_mean_p || !d_losses || !d_n_valid)
        return fail("balance: null pointer");
    if (logits_stride % 4 || logits_stride < (size_t)n_experts * 4)
        return fail("balance: logits stride %zu below a row of %d floats, or no multiple of 4", logits_stride, n_experts);
    const BalanceSpace sp = balance_space(n_tokens, n_experts, n_groups);
    if (!d_workspace || workspace_bytes < sp.bytes || (uintptr_t)d_workspace % 16)
        return fail("balance: the workspace must be 16-byte aligned and hold %zu bytes (got %zu)", sp.bytes, workspace_bytes);
    if (g_device < 0) return fail("sabah_rt_init has not been called");
    if (!check_sticky()) return -1;
    OnDevice dev;
    if (!dev.ok) return -1;
    uint8_t* ws = static_cast<uint8_t*>(d_workspace);
    BalanceArgs a{};
    a.logits = reinterpret_cast<const uint8_t*>(d_logits);
    a.stride = logits_stride;
    a.ids = d_ids;
    a.mask = d_mask;
    a.n_experts = n_experts;
    a.n_used = n_used;
    a.n_groups = n_groups;
    a.group_len = n_tokens / n_groups;
    balance_plan(n_tokens, n_groups, a.chunks, a.chunk_len);
    a.part_p = reinterpret_cast<float*>(ws + sp.p);
    a.part_c = reinterpret_cast<int*>(ws + sp.c);
    a.part_z = reinterpret_cast<float2*>(ws + sp.z);
    a.part_loss = reinterpret_cast<double*>(ws + sp.loss);
    a.group = reinterpret_cast<double2*>(ws + sp.group);
    a.ticket = reinterpret_cast<unsigned*>(ws + sp.ticket);
    a.counts = d_counts;
    a.mean_p = d_mean_p;
    a.losses = d_losses;
    a.n_valid = d_n_valid;
    a.err = g_err_dev;
    hipStream_t st = pick_stream(stream);
    if (n_experts <= 64) launch_balance_rows<1, 1, 1>(a, st);
    else if (n_experts <= 128) launch_balance_rows<2, 2, 1>(a, st);
    else if (n_experts <= 256) launch_balance_rows<4, 4, 1>(a, st);
    else if (n_experts <= 512) launch_balance_rows<8, 4, 1>(a, st);
    else if (n_experts <= 2048) launch_balance_rows<8, 4, 4>(a, st);
    else launch_balance_rows<8, 4, 8>(a, st);
    if (!ck(hipGetLastError(), "balance launch")) return -1;
    hipLaunchKernelGGL(k_balance_sum, dim3((unsigned)((n_experts + kBalanceCols - 1) / kBalanceCols), (unsigned)n_groups),
                       dim3(kBalanceSumThreads), 0, st, a);
    return ck(hipGetLastError(), "balance sum launch") ? 0 : -1;
}

template <int PER, int VEC, int W>
static void launch_route_backward(const RouteBackArgs& a, hipStream_t st) {
    constexpr int kSide = row_threads(W) / (64 * W);               // tokens of a workgroup
    // a launch takes fewer than 2^32 threads along x, and 2^24 tokens of a workgroup each are more
    constexpr unsigned kMost = 1u << 20;
    const unsigned groups = (unsigned)((a.n_tokens + kSide - 1) / kSide);
    hipLaunchKernelGGL((k_route_backward<PER, VEC, W>), dim3(std::min(groups, kMost), (groups + kMost - 1) / kMost),
                       dim3(row_threads(W)), 0, st, a);
}

SABAH_API int sabah_moe_route_backward(const float* d_logits, size_t logits_stride, const int32_t* d_ids,
                                       const uint8_t* d_mask, int n_tokens, int n_experts, int n_used, int norm_w,
                                       float w_scale, const float* d_dw, const int32_t* d_counts,
                                       const int32_t* d_n_valid, int n_groups, float c_balance, float c_z,
                                       float* d_dlogits, size_t dlogits_stride, void* stream) {
    if (check_router_shape("route backward", n_tokens, n_experts, n_used, n_groups)) return -1;
    if (n_tokens && (!d_logits || !d_dlogits || (!d_ids && d_dw))) return fail("route backward: null pointer");
    if (!(w_scale > 0.0f) || w_scale == __builtin_inff())
        return fail("route backward: w_scale must be positive and finite");
    const bool losses = c_balance != 0.0f || c_z != 0.0f;
    if (losses && (!d_counts || !d_n_valid))
        return fail("route backward: a loss's gradient needs the counts and n_valid of sabah_moe_balance");
    if (logits_stride % 4 || dlogits_stride % 4 || logits_stride < (size_t)n_experts * 4 ||
        dlogits_stride < (size_t)n_experts * 4)
        return fail("route backward: a stride (%zu, %zu) below a row of %d floats, or no multiple of 4", logits_stride,
                    dlogits_stride, n_experts);
    if (g_device < 0) return fail("sabah_rt_init has not been called");
    if (!check_sticky()) return -1;
    if (n_tokens == 0) return 0;
    OnDevice dev;
    if (!dev.ok) return -1;
    RouteBackArgs a{};
    a.logits = reinterpret_cast<const uint8_t*>(d_logits);
    a.stride = logits_stride;
    a.ids = d_ids;
    a.mask = d_mask;
    a.dw = d_dw;
    a.counts = losses ? d_counts : nullptr;
    a.n_valid = d_n_valid;
    a.dlogits = reinterpret_cast<uint8_t*>(d_dlogits);
    a.dstride = dlogits_stride;
    a.n_tokens = n_tokens;
    a.n_experts = n_experts;
    a.n_used = n_used;
    a.norm_w = norm_w ? 1 : 0;
    a.n_groups = n_groups;
    a.group_len = n_tokens / n_groups;
    a.w_scale = w_scale;
    a.c_balance = c_balance;
    a.c_z = c_z;
    a.err = g_err_dev;
    hipStream_t st = pick_stream(stream);
    if (n_experts <= 64) launch_route_backward<1, 1, 1>(a, st);
    else if (n_experts <= 128) launch_route_backward<2, 2, 1>(a, st);
    else if (n_experts <= 256) launch_route_backward<4, 4, 1>(a, st);
    else if (n_experts <= 512) launch_route_backward<8, 4, 1>(a, st);
    else if (n_experts <= 2048) launch_route_backward<8, 4, 4>(a, st);
    else launch_route_backward<8, 4, 8>(a, st);
    return ck(hipGetLastError(), "route backward launch") ? 0 : -1;
}

// ---------------------------------------------------------------------------
// adapters
// ---------------------------------------------------------------------------
template <int NR, int H>
constexpr int kLoraExpandOcc = NR * H <= 2 ? 3 : NR <= 4 ? 2 : 1;   // waves per SIMD that the registers are kept to

// type codes of adapter weights (ggml's F32, F16 and BF16)
constexpr int kLoraMaxKeys = 1 << 21;         // (adapter, expert) pairs: a key and its row sort as one 32-bit word
constexpr int kTypeF32 = 0, kTypeF16 = 1, kTypeBF16 = 30;

static int check_lora(const char* what, const sabah_lora_desc* L, int n_ids, int n_tokens) {
    if (!L || !L->a || !L->b) return fail("%s: null adapter bank", what);
    if (L->type != kTypeF32 && L->type != kTypeF16 && L->type != kTypeBF16)
        return fail("%s: adapter type %d is none of F32 (0), F16 (1), BF16 (30)", what, L->type);
    if (L->rank <= 0 || L->rank > kLoraMaxRank) return fail("%s: rank %d outside [1, %d]", what, L->rank, kLoraMaxRank);
    if (L->n_adapters <= 0 || L->n_experts <= 0 || L->k <= 0 || L->rows <= 0 ||
        (long long)L->n_adapters * L->n_experts > kLoraMaxKeys || (long long)L->rank * L->k > 1 << 28 || (long long)L->rank * L->rows > 1 << 28)
        return fail("%s: invalid geometry (n_adapters=%d n_experts=%d k=%d rows=%d)", what, L->n_adapters, L->n_experts,
                    L->k, L->rows);
    if (n_ids <= 0 || n_tokens < 0 || (long long)n_ids * n_tokens > 1 << 24)
        return fail("%s: n_ids=%d, n_tokens=%d give no rows, or too many", what, n_ids, n_tokens);
    return 0;
}

static bool stride_ok(size_t s) { return s % 4 == 0; }

// Forward.  A call of at most kLoraDirectRows rows is one launch (k_lora_apply): at 256 rows of 64 adapters (k 2048, rows
// 512, rank 16, the one shape timed) 16.2 us, where the three launches of a larger call take 20.2 (15.6 and 16.4 at 128, 14.9
// and 15.8 at 64).
// Above, each window of rows has at most one tile per 16 rows and one more per key.  With kLoraFusedTiles of them, two
// for every CU, a workgroup shrinks and expands its tile (one launch after the lists); with fewer two launches share out k and the
// columns.  us of the one launch against the two, 2048 x 2048, rank 32, 8 adapters: 44.8 and 36.0 at 4,096 rows (328 tiles),
// 56.2 and 59.0 at 8,192 (656), 95.3 and 103.5 at 16,384; of 512 experts' pairs 14.7 and 17.0 at 640 rows, 21.0 and 30.9 at 5,120.
constexpr int kLoraDirectRows = 256;
constexpr int kLoraFusedTiles = 512;
// The two launches: k in parts of at least eight steps of 32, up to about 1,024 workgroups (1,999 rows of k 2048 at rank 64: the
// shrink 12.4 us in eight parts, 25.8 whole; the expand, which adds them up, 11.2 and 8.4)
constexpr int kLoraShrinkGroups = 1024, kLoraShrinkParts = 8, kLoraShrinkSteps = 8;
// Of a k of at least parts * kLoraShrinkSteps steps, the last part has at least kLoraShrinkSteps + 2 - parts.  It has to have two:
// LoraShrink gives k's rest to the part whose whole steps end there, which two would be if the last were that rest alone.
static_assert(kLoraShrinkSteps >= kLoraShrinkParts, "a last part of k's rest alone would be summed twice");
constexpr int kLoraExpandGroups = 1024;
// k of a shrink in parts while there are few tiles
static void lora_k_parts(int k, int tiles, int& parts, int& steps) {
    const int all = (k + 31) / 32;
    parts = std::max(1, std::min({kLoraShrinkParts, kLoraShrinkGroups / tiles, all / kLoraShrinkSteps}));
    steps = (all + parts - 1) / parts;
    parts = (all + steps - 1) / steps;
}

// The expand's columns in parts of a step of 64 or more for each of its four waves, about kLoraExpandGroups workgroups
static int lora_columns(int columns, int tiles, int& cols) {
    const int parts = std::max(1, std::min((columns + 255) / 256, kLoraExpandGroups / tiles));
    cols = ((columns + parts - 1) / parts + 63) / 64 * 64;
    return (columns + cols - 1) / cols;
}

struct LoraSpace {
    size_t order, items, n_items, s, bytes;
    int windows, slots, key_bits, k_parts, k_steps, rank16;
};
static LoraSpace lora_space(const sabah_lora_desc* L, int n_rows) {
    LoraSpace s{};
    const int keys = L->n_adapters * L->n_experts + 2;      // without an adapter, and with a bad id
    const int span = std::min(n_rows, kLoraWindow);
    s.windows = (n_rows + kLoraWindow - 1) / kLoraWindow;
    s.slots = std::min(span, span / kLoraTile + std::min(keys, span));
    s.rank16 = L->rank <= 16 ? 16 : L->rank <= 32 ? 32 : L->rank <= 64 ? 64 : 128;
    while (keys >> s.key_bits) ++s.key_bits;                // the word past the rows has key + 2 == keys
    if (n_rows <= kLoraDirectRows) {
        s.windows = 1;
        return s;
    }
    lora_k_parts(L->k, (n_rows + kLoraTile - 1) / kLoraTile, s.k_parts, s.k_steps);
    const size_t positions = (long long)s.windows * s.slots < kLoraFusedTiles ? (size_t)s.windows * kLoraWindow : 0;
    s.items = align256((size_t)s.windows * kLoraWindow * 4);
    s.n_items = s.items + align256((size_t)s.windows * s.slots * 16);
    s.s = s.n_items + align256((size_t)s.windows * 4);
    s.bytes = s.s + align256(s.k_parts * positions * s.rank16 * 4);
    if (!positions) s.s = 0;
    return s;
}

// A backward call's: the tiles and runs, s and u, the transposed pairs, the pieces and offsets that
// the weights' gradients read, and their partial sums.
struct LoraBackSpace {
    size_t order, items, n_items, runs, s, u, at, bt, ps, pu, ox, oy, part, bytes;
    int windows, slots, key_bits, rank16, positions, tiles_a, tiles_b, splits;
};
// Rows up to which a workgroup of the backward's shrinks takes half a tile, with eight waves.  A CU reads its tile's rows
// and A at little more than 64 bytes a cycle, so few tiles are shared out; many read A half as often as wholes.  us at 512 /
// 1,024 / 2,048 rows, k 2048, halves against wholes: f32 to 768 at rank 16 8.1 / 8.9 / 11.7 against 13.3 / 14.2 / 15.6,
// bf16 to 2048 at rank 64 11.3 / 11.9 / 18.6 against 21.4 / 22.0 / 22.5.  At 8,192 the latter takes 55 - 65 in halves, 52 in
// wholes: the crossing lies between, where nothing was timed
constexpr int kLoraHalfRows = 2048;
constexpr int kLoraBackKeys = 1 << 15;        // a word per key and window
// Splits of the weights' gradients, over the windows: what one request sends is together, so without them the
// longest request's key would be a few workgroups' work
constexpr int kLoraGradSplits = 8;
constexpr size_t kLoraGradBytes = (size_t)128 << 20;    // of partial sums at most
static LoraBackSpace lora_back_space(const sabah_lora_desc* L, int n_rows) {
    LoraBackSpace s{};
    const int keys = L->n_adapters * L->n_experts, span = std::min(n_rows, kLoraWindow);
    s.windows = std::max(1, (n_rows + kLoraWindow - 1) / kLoraWindow);
    s.slots = std::max(1, std::min(span, span / 32 + std::min(keys + 2, span)));
    s.rank16 = L->rank <= 16 ? 16 : L->rank <= 32 ? 32 : L->rank <= 64 ? 64 : 128;
    while ((keys + 2) >> s.key_bits) ++s.key_bits;
    s.positions = s.windows * kLoraWindow;
    s.tiles_a = (L->k + 63) / 64;
    s.tiles_b = (L->rows + 63) / 64;
    const size_t part = (size_t)keys * (s.tiles_a + s.tiles_b) * s.rank16 * 64 * 4;
    s.splits = (int)std::max<size_t>(1, std::min<size_t>({(size_t)s.windows, (size_t)kLoraGradSplits, kLoraGradBytes / part}));
    const size_t esize = L->type == kTypeF32 ? 4 : 2, all = (size_t)s.windows * s.slots;
    size_t at = 0;
    auto take = [&](size_t n) {
        const size_t here = at;
        at += align256(n);
        return here;
    };
    s.order = take((size_t)s.positions * 4);
    s.items = take(all * 16);
    s.n_items = take((size_t)s.windows * 4);
    s.runs = take((size_t)s.windows * keys * 4);
    s.s = take((size_t)s.positions * s.rank16 * 4);
    s.u = take((size_t)s.positions * s.rank16 * 4);
    s.at = take((size_t)keys * L->rank * L->k * esize);
    s.bt = take((size_t)keys * L->rank * L->rows * esize);
    s.ps = take(all * 3 * s.rank16 * 64);
    s.pu = take(all * 3 * s.rank16 * 64);
    s.ox = take(all * 32 * 8);
    s.oy = take(all * 32 * 8);
    s.part = take(s.splits > 1 ? s.splits * part : 0);
    s.bytes = at;
    return s;
}

static int check_lora_keys(const sabah_lora_desc* L) {
    if ((long long)L->n_adapters * L->n_experts > kLoraBackKeys)
        return fail("adapters backward: %d adapters of %d experts are more than %d pairs", L->n_adapters, L->n_experts,
                    kLoraBackKeys);
    return 0;
}

SABAH_API size_t sabah_lora_workspace(const sabah_lora_desc* lora, int n_ids, int n_tokens, int backward) {
    if (check_lora("adapters", lora, n_ids, n_tokens) || (backward && check_lora_keys(lora))) return 0;
    return backward ? lora_back_space(lora, n_ids * n_tokens).bytes : lora_space(lora, n_ids * n_tokens).bytes;
}

static LoraArgs lora_args(const sabah_lora_desc* L, const float* d_x, size_t x_id_stride, int x_rows,
                          size_t x_token_stride, const int32_t* d_adapters, const int32_t* d_ids, size_t ids_id_stride,
                          size_t ids_token_stride, int n_ids, int n_tokens) {
    LoraArgs a{};
    a.x = reinterpret_cast<const uint8_t*>(d_x);
    a.x_id = x_id_stride;
    a.x_tok = x_token_stride;
    a.x_rows = x_rows;
    a.adapters = d_adapters;
    a.ids = reinterpret_cast<const uint8_t*>(d_ids);
    a.ids_id = ids_id_stride;
    a.ids_tok = ids_token_stride;
    a.n_ids = n_ids;
    a.n_tokens = n_tokens;
    a.a = L->a;
    a.b = L->b;
    a.scale = L->scale;
    a.ranks = L->ranks;
    a.n_adapters = L->n_adapters;
    a.n_experts = L->n_experts;
    a.rank = L->rank;
    a.k = L->k;
    a.rows = L->rows;
    a.err = g_err_dev;
    return a;
}

static int check_lora_rows(const char* what, const sabah_lora_desc* L, const float* d_x, size_t x_id_stride, int x_rows,
                           size_t x_token_stride, const int32_t* d_adapters, const int32_t* d_ids, size_t ids_id_stride,
                           size_t ids_token_stride, int n_ids, int n_tokens) {
    if (check_lora(what, L, n_ids, n_tokens)) return -1;
    if (n_tokens && (!d_x || !d_adapters)) return fail("%s: null pointer", what);
    if (!d_ids && L->n_experts != 1) return fail("%s: %d experts need ids", what, L->n_experts);
    if (x_rows != 1 && x_rows != n_ids) return fail("%s: %d input rows, expected 1 or n_ids=%d", what, x_rows, n_ids);
    if (!stride_ok(x_id_stride) || !stride_ok(x_token_stride) || !stride_ok(ids_id_stride) || !stride_ok(ids_token_stride))
        return fail("%s: strides are in bytes and multiples of 4", what);
    return 0;
}

template <typename W, int NR, int NW, int US, int U, int OCC>
static void launch_lora_apply_rank(const LoraArgs& a, const LoraTiles& t, int column_parts, int windows, hipStream_t st) {
    const dim3 grid((unsigned)t.slots, (unsigned)column_parts, (unsigned)windows);
    if (!t.order) {
        hipLaunchKernelGGL((k_lora_apply<W, NR, NW, US, 1, true>), grid, dim3(64 * NW), 0, st, a, t);
        return;
    }
    if (!t.s) {
        hipLaunchKernelGGL((k_lora_apply<W, NR, 4, U, OCC, false>), grid, dim3(256), 0, st, a, t);
        return;
    }
    hipLaunchKernelGGL((k_lora_shrink<W, NR, 4, U, OCC, 1, false>), dim3((unsigned)t.slots, (unsigned)t.k_parts, (unsigned)windows),
                       dim3(256), 0, st, a, t, a, t, windows);
    hipLaunchKernelGGL((k_lora_expand<W, NR, kLoraExpandOcc<NR, 1>, 1>), grid, dim3(256), 0, st, a, t);
}
template <typename W>
static void launch_lora_apply(const LoraArgs& a, const LoraTiles& t, int column_parts, int windows, hipStream_t st) {
    if (a.rank <= 16) launch_lora_apply_rank<W, 1, 8, 4, 2, 4>(a, t, column_parts, windows, st);
    else if (a.rank <= 32) launch_lora_apply_rank<W, 2, 8, 4, 2, 4>(a, t, column_parts, windows, st);
    else if (a.rank <= 64) launch_lora_apply_rank<W, 4, 4, 2, 2, 2>(a, t, column_parts, windows, st);
    else launch_lora_apply_rank<W, 8, 4, 1, 1, sizeof(typename W::T) == 4 ? 1 : 2>(a, t, column_parts, windows, st);
}

SABAH_API int sabah_lora_apply(const sabah_lora_desc* lora, const float* d_x, size_t x_id_stride, int x_rows,
                               size_t x_token_stride, const int32_t* d_adapters, const int32_t* d_ids,
                               size_t ids_id_stride, size_t ids_token_stride, int n_ids, int n_tokens,
                               const float* d_base, size_t base_id_stride, size_t base_token_stride, float* d_dst,
                               size_t dst_id_stride, size_t dst_token_stride, void* d_workspace, size_t workspace_bytes,
                               void* stream) {
    if (check_lora_rows("adapters", lora, d_x, x_id_stride, x_rows, x_token_stride, d_adapters, d_ids, ids_id_stride,
                        ids_token_stride, n_ids, n_tokens))
        return -1;
    if (n_tokens && !d_dst) return fail("adapters: null pointer");
    if (!stride_ok(base_id_stride) || !stride_ok(base_token_stride) || !stride_ok(dst_id_stride) ||
        !stride_ok(dst_token_stride))
        return fail("adapters: strides are in bytes and multiples of 4");
    // a stride that no row is reached by may be anything
    if (d_base == d_dst && ((n_ids > 1 && base_id_stride != dst_id_stride) || (n_tokens > 1 && base_token_stride != dst_token_stride)))
        return fail("adapters: base in place of dst needs dst's strides");
    const int n_rows = n_ids * n_tokens;
    const LoraSpace sp = lora_space(lora, n_rows);
    if (sp.bytes && (!d_workspace || workspace_bytes < sp.bytes || (uintptr_t)d_workspace % 16))
        return fail("adapters: the workspace must be 16-byte aligned and hold %zu bytes (got %zu)", sp.bytes,
                    workspace_bytes);
    if (g_device < 0) return fail("sabah_rt_init has not been called");
    if (n_tokens && d_dst == d_x) return fail("adapters: dst would overwrite x");
    if (!check_sticky()) return -1;
    if (n_tokens == 0) return 0;
    OnDevice dev;
    if (!dev.ok) return -1;
    LoraArgs a = lora_args(lora, d_x, x_id_stride, x_rows, x_token_stride, d_adapters, d_ids, ids_id_stride,
                           ids_token_stride, n_ids, n_tokens);
    a.base = reinterpret_cast<const uint8_t*>(d_base);
    a.base_id = base_id_stride;
    a.base_tok = base_token_stride;
    a.dst = reinterpret_cast<uint8_t*>(d_dst);
    a.dst_id = dst_id_stride;
    a.dst_tok = dst_token_stride;
    hipStream_t st = pick_stream(stream);
    LoraTiles t{};
    t.n_rows = n_rows;
    t.slots = sp.slots;
    t.skip_none = d_base == d_dst;
    t.key_bits = sp.key_bits;
    if (sp.bytes) {
        uint8_t* ws = static_cast<uint8_t*>(d_workspace);
        const LoraGroup g{reinterpret_cast<int*>(ws + sp.order), reinterpret_cast<int4*>(ws + sp.items),
                          reinterpret_cast<int*>(ws + sp.n_items), n_rows, sp.slots, t.skip_none, sp.key_bits, kLoraTile, nullptr};
        hipLaunchKernelGGL(k_lora_group, dim3((unsigned)sp.windows),
                           dim3((unsigned)std::min(kLoraWindow, (n_rows + 63) / 64 * 64)), 0, st, a, g);
        if (!ck(hipGetLastError(), "adapters grouping launch")) return -1;
        t.order = g.order;
        t.items = g.items;
        t.n_items = g.n_items;
        t.s = sp.s ? reinterpret_cast<float*>(ws + sp.s) : nullptr;
        t.k_parts = sp.k_parts;
        t.k_steps = sp.k_steps;
        t.positions = sp.windows * kLoraWindow;
    }
    int parts = 1;
    t.cols = (lora->rows + 63) / 64 * 64;
    if (t.s) {
        parts = lora_columns(lora->rows, (n_rows + kLoraTile - 1) / kLoraTile, t.cols);
    } else if (!sp.bytes) {                                 // what fills the chip
        parts = std::max(1, std::min((lora->rows + 63) / 64, 2 * g_num_cu / sp.slots));
        t.cols = ((lora->rows + parts - 1) / parts + 63) / 64 * 64;
        parts = (lora->rows + t.cols - 1) / t.cols;
    }
    switch (lora->type) {
    case kTypeF32: launch_lora_apply<LoraF32>(a, t, parts, sp.windows, st); break;
    case kTypeF16: launch_lora_apply<LoraF16>(a, t, parts, sp.windows, st); break;
    default: launch_lora_apply<LoraBF16>(a, t, parts, sp.windows, st); break;
    }
    return ck(hipGetLastError(), "adapters launch") ? 0 : -1;
}

struct LoraBack {
    LoraBackSpace sp;
    LoraArgs a, u, x;             // s = A x; u = c B^T dy; dx = A^T u
    LoraGroup g;
    LoraTiles ts, tu;
    LoraTurn turn;
    LoraGrad w;
    int grad_tiles;
    hipStream_t st;
};

template <typename W, int NR, int U, int OCC, int GOCC>
static int launch_lora_back_rank(const LoraBack& b) {
    const LoraBackSpace& sp = b.sp;
    const unsigned slots = (unsigned)sp.slots, windows = (unsigned)sp.windows, keys = (unsigned)b.w.keys;
    hipLaunchKernelGGL(k_lora_group, dim3(windows), dim3((unsigned)std::max(64, std::min(kLoraWindow, (b.g.n_rows + 63) / 64 * 64))),
                       0, b.st, b.a, b.g);
    if (b.g.n_rows && (b.x.dst || b.grad_tiles)) {
        hipLaunchKernelGGL(k_lora_transpose<typename W::T>, dim3((unsigned)(sp.tiles_a + sp.tiles_b), keys), dim3(256), 0, b.st, b.turn);
        const unsigned sides = windows * (b.grad_tiles ? 2u : 1u);
        if (b.g.n_rows <= kLoraHalfRows)
            hipLaunchKernelGGL((k_lora_shrink<W, NR, 8, U, 1, 1, true>), dim3(slots, 2u, sides), dim3(512), 0, b.st, b.u, b.tu, b.a, b.ts, (int)windows);
        else
            hipLaunchKernelGGL((k_lora_shrink<W, NR, 4, U, OCC, 2, false>), dim3(slots, 1u, sides), dim3(256), 0, b.st, b.u, b.tu, b.a, b.ts, (int)windows);
    }
    if (b.g.n_rows && b.x.dst) {
        LoraTiles t = b.tu;
        const int parts = lora_columns(b.x.rows, (b.g.n_rows + 31) / 32, t.cols);
        hipLaunchKernelGGL((k_lora_expand<W, NR, kLoraExpandOcc<NR, 2>, 2>), dim3(slots, (unsigned)parts, windows), dim3(256), 0, b.st, b.x, t);
    }
    if (b.grad_tiles) {
        hipLaunchKernelGGL((k_lora_grad<NR, GOCC>), dim3((unsigned)b.grad_tiles, keys, (unsigned)b.w.splits), dim3(256), 0, b.st, b.w);
        if (b.w.splits > 1)
            hipLaunchKernelGGL(k_lora_grad_sum<NR>, dim3((unsigned)b.grad_tiles, keys, (unsigned)((b.a.rank + 15) / 16)), dim3(256), 0, b.st, b.w);
    }
    return ck(hipGetLastError(), "adapters backward launch") ? 0 : -1;
}
template <typename W>
static int launch_lora_back(const LoraBack& b) {
    if (b.a.rank <= 16) return launch_lora_back_rank<W, 1, 2, 3, 3>(b);
    if (b.a.rank <= 32) return launch_lora_back_rank<W, 2, 2, 3, 2>(b);
    if (b.a.rank <= 64) return launch_lora_back_rank<W, 4, 1, 2, 2>(b);
    return launch_lora_back_rank<W, 8, 1, 1, 1>(b);
}

SABAH_API int sabah_lora_backward(const sabah_lora_desc* lora, const float* d_x, size_t x_id_stride, int x_rows,
                                  size_t x_token_stride, const int32_t* d_adapters, const int32_t* d_ids,
                                  size_t ids_id_stride, size_t ids_token_stride, int n_ids, int n_tokens,
                                  const float* d_dy, size_t dy_id_stride, size_t dy_token_stride, float* d_dx,
                                  size_t dx_id_stride, size_t dx_token_stride, int add_dx, float* d_da, float* d_db,
                                  int add_dw, void* d_workspace, size_t workspace_bytes, void* stream) {
    if (check_lora_rows("adapters backward", lora, d_x, x_id_stride, x_rows, x_token_stride, d_adapters, d_ids,
                        ids_id_stride, ids_token_stride, n_ids, n_tokens))
        return -1;
    if (n_tokens && !d_dy) return fail("adapters backward: null pointer");
    if (!stride_ok(dy_id_stride) || !stride_ok(dy_token_stride) || !stride_ok(dx_id_stride) || !stride_ok(dx_token_stride))
        return fail("adapters backward: strides are in bytes and multiples of 4");
    if (check_lora_keys(lora)) return -1;
    const int n_rows = n_ids * n_tokens, keys = lora->n_adapters * lora->n_experts;
    const LoraBackSpace sp = lora_back_space(lora, n_rows);
    if (!d_workspace || workspace_bytes < sp.bytes || (uintptr_t)d_workspace % 16)
        return fail("adapters backward: the workspace must be 16-byte aligned and hold %zu bytes (got %zu)", sp.bytes,
                    workspace_bytes);
    if (g_device < 0) return fail("sabah_rt_init has not been called");
    if (n_tokens && d_dx && (d_dx == d_x || d_dx == d_dy)) return fail("adapters backward: dx would overwrite x or dy");
    if (!check_sticky()) return -1;
    OnDevice dev;
    if (!dev.ok) return -1;
    LoraArgs a = lora_args(lora, d_x, x_id_stride, x_rows, x_token_stride, d_adapters, d_ids, ids_id_stride,
                           ids_token_stride, n_ids, n_tokens);
    a.dy = reinterpret_cast<const uint8_t*>(d_dy);
    a.dy_id = dy_id_stride;
    a.dy_tok = dy_token_stride;
    uint8_t* ws = static_cast<uint8_t*>(d_workspace);
    LoraBack b{};
    b.sp = sp;
    b.st = pick_stream(stream);
    b.a = a;
    b.u = a;                                                // u: dy shrunk by B^T
    b.u.x = a.dy;
    b.u.x_id = dy_id_stride;
    b.u.x_tok = dy_token_stride;
    b.u.x_rows = n_ids;
    b.u.k = lora->rows;
    b.u.a = ws + sp.bt;
    b.x = a;                                                // dx: u expanded by A^T
    b.x.b = ws + sp.at;
    b.x.rows = lora->k;
    b.x.dst = reinterpret_cast<uint8_t*>(d_dx);
    b.x.dst_id = dx_id_stride;
    b.x.dst_tok = dx_token_stride;
    b.x.base = add_dx ? b.x.dst : nullptr;
    b.x.base_id = dx_id_stride;
    b.x.base_tok = dx_token_stride;
    const LoraGroup g{reinterpret_cast<int*>(ws + sp.order), reinterpret_cast<int4*>(ws + sp.items),
                      reinterpret_cast<int*>(ws + sp.n_items), n_rows, sp.slots, !d_dx || add_dx, sp.key_bits, 32,
                      reinterpret_cast<uint32_t*>(ws + sp.runs)};
    b.g = g;
    LoraTiles t{};
    t.order = g.order;
    t.items = g.items;
    t.n_items = g.n_items;
    t.n_rows = n_rows;
    t.slots = sp.slots;
    t.skip_none = g.skip_none;
    t.key_bits = sp.key_bits;
    t.positions = sp.positions;
    b.ts = b.tu = t;
    b.ts.s = reinterpret_cast<float*>(ws + sp.s);
    b.ts.k_parts = 1;                                       // whole: the epilogue writes the pieces
    b.ts.k_steps = (lora->k + 31) / 32;
    b.ts.pieces = reinterpret_cast<uint16_t*>(ws + sp.ps);
    b.ts.off = reinterpret_cast<uint64_t*>(ws + sp.ox);
    b.tu.s = reinterpret_cast<float*>(ws + sp.u);
    b.tu.k_parts = 1;
    b.tu.k_steps = (lora->rows + 31) / 32;
    b.tu.pieces = d_da || d_db ? reinterpret_cast<uint16_t*>(ws + sp.pu) : nullptr;
    b.tu.off = reinterpret_cast<uint64_t*>(ws + sp.oy);
    b.tu.scaled = 1;
    b.turn = LoraTurn{lora->a, lora->b, ws + sp.at, ws + sp.bt, g.runs, sp.windows, keys, lora->rank, lora->k, lora->rows,
                      sp.tiles_a};
    LoraGrad& w = b.w;
    w.runs = g.runs;
    w.windows = sp.windows;
    w.keys = keys;
    w.slots = sp.slots;
    w.splits = sp.splits;
    w.rank = lora->rank;
    w.tiles_a = d_da ? sp.tiles_a : 0;
    w.p[0] = reinterpret_cast<const uint16_t*>(ws + sp.pu);
    w.p[1] = b.ts.pieces;
    w.off[0] = b.ts.off;
    w.off[1] = b.tu.off;
    w.src[0] = a.x;
    w.src[1] = a.dy;
    w.width[0] = lora->k;
    w.width[1] = lora->rows;
    w.out[0] = d_da;
    w.out[1] = d_db;
    w.part[0] = reinterpret_cast<float*>(ws + sp.part);
    w.part[1] = w.part[0] + (size_t)sp.splits * keys * sp.tiles_a * sp.rank16 * 64;
    w.scale = lora->scale;
    w.ranks = lora->ranks;
    w.n_experts = lora->n_experts;
    w.add = add_dw != 0;
    b.grad_tiles = w.tiles_a + (d_db ? sp.tiles_b : 0);
    switch (lora->type) {
    case kTypeF32: return launch_lora_back<LoraF32>(b);
    case kTypeF16: return launch_lora_back<LoraF16>(b);
    default: return launch_lora_back<LoraBF16>(b);
    }
}
