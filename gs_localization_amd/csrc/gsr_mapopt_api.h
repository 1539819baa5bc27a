// gsr_mapopt_api.h -- host side of gsr_mapopt.h: checks of arguments, tables of a launch, launches.  Part of gsr_api.hip (fail,
// select_device_of, Carver are its own); the C entry points are there.
#pragma once

namespace {
static_assert(sizeof(gsr::OptArgs) <= 4096 && sizeof(gsr::RowArgs) <= 4096 && sizeof(gsr::NormArgs) <= 4096 && sizeof(gsr::MomentArgs) <= 4096,
              "a launch's table must fit the kernel arguments");
// Of one tensor.  A launch has under 2^32 threads, so under 2^24 workgroups of 4096 elements; a call writes all its memory once, at least six
// bytes for an element, so the card's 288 GB hold no more.
const long long kOptMaxElements = 1LL << 35;
const int kOptGrid = 2048;                            // workgroups of the norm's launches: eight per CU, each walks chunks
// Past the caches (opt_get) from 256 MB on, what lies behind the L2; `bytes` counts what a step reads.  32-bit moments, cached / past the caches, a step
// that follows its like: 128 MB 38 / 43 us, 256 71 / 81, 320 95 / 103, 384 135 / 122, 640 222 / 199; behind a GB of other work, as in a
// training step: 62 / 48, 105 / 84, 128 / 106, 146 / 125, 231 / 201 (8 bits alike: 40 / 42, 72 / 78, 91 / 95, 119 / 112, 204 / 180).
bool opt_stream(long long bytes) { return bytes > 256LL << 20; }
bool opt_type_ok(int t) { return t == GSR_TYPE_F32 || t == GSR_TYPE_BF16 || t == GSR_TYPE_F16; }
long long opt_size(int t) { return t == GSR_TYPE_F32 ? 4 : 2; }
bool opt_aligned(const void* p, long long element) { return ((uintptr_t)p & (uintptr_t)(4 * element - 1)) == 0; }          // to four elements
int opt_grid(uint32_t chunks) { return (int)std::max<uint32_t>(1u, std::min<uint32_t>(chunks, (uint32_t)kOptGrid)); }

// Memory that one call writes: no two ranges of it, and no range that it only reads, may overlap.
struct OptRanges {
    struct R { uintptr_t lo, hi; bool write; };
    std::vector<R> r;
    void add(const void* p, long long bytes, bool write) { if (p && bytes > 0) r.push_back({(uintptr_t)p, (uintptr_t)p + (uintptr_t)bytes, write}); }
    bool clash()
    {
        std::sort(r.begin(), r.end(), [](const R& a, const R& b) { return a.lo < b.lo; });
        uintptr_t end = 0, wend = 0;          // of everything so far, and of what is written
        for (const R& x : r) {
            if (x.lo < wend || (x.write && x.lo < end)) return true;
            end = std::max(end, x.hi);
            if (x.write) wend = std::max(wend, x.hi);
        }
        return false;
    }
};

// The largest |m| / sqrt(v) that gradients can bring about: the 8-bit ratio has 127 steps of it to either side.
bool opt_spannable(double beta1, double beta2) { return beta1 >= 0.0 && beta1 * beta1 < beta2 && beta2 < 1.0; }
double opt_span(double beta1, double beta2) { return (1.0 - beta1) / sqrt((1.0 - beta2) * (1.0 - beta1 * beta1 / beta2)); }

int adamw_check(const gsr_adamw_args* a, const gsr_code_origin* origins)
{
    if (a->n_tensors < 0 || (a->n_tensors > 0 && !a->tensors)) return fail(GSR_E_INVALID, "gsr_adamw_step: NULL pointer%s", "");
    if (a->state_bits != 32 && a->state_bits != 8) return fail(GSR_E_INVALID, "gsr_adamw_step: moments have 32 or 8 bits%s", "");
    if (!(a->beta1 >= 0.0 && a->beta1 < 1.0 && a->beta2 >= 0.0 && a->beta2 < 1.0)) return fail(GSR_E_INVALID, "gsr_adamw_step: 0 <= beta < 1 required%s", "");
    if (!(a->eps >= 0.0)) return fail(GSR_E_INVALID, "gsr_adamw_step: eps >= 0 required%s", "");
    const bool eight = a->state_bits == 8;
    if (eight && !opt_spannable(a->beta1, a->beta2)) return fail(GSR_E_INVALID, "gsr_adamw_step: 8-bit moments need beta1^2 < beta2 (otherwise m / sqrt(v) has no bound)%s", "");
    OptRanges ranges;
    ranges.r.reserve((size_t)a->n_tensors * 6 + 1);
    for (int i = 0; i < a->n_tensors; i++) {
        const gsr_opt_tensor& t = a->tensors[i];
        if (t.n < 0 || t.n > kOptMaxElements) return fail(GSR_E_INVALID, "gsr_adamw_step: bad tensor size%s", "");
        if (!opt_type_ok(t.param_type) || !opt_type_ok(t.grad_type)) return fail(GSR_E_INVALID, "gsr_adamw_step: unknown type%s", "");
        if (eight && origins && !opt_spannable(origins[i].beta1, origins[i].beta2))
            return fail(GSR_E_INVALID, "gsr_adamw_step: the betas of a tensor's codes: 0 <= beta1, beta1^2 < beta2 < 1 required%s", "");
        if (!t.clock || (t.n > 0 && (!t.param || !t.grad || !t.state0 || !t.state1 || (eight && !t.window))))
            return fail(GSR_E_INVALID, "gsr_adamw_step: NULL pointer%s", "");
        if (((uintptr_t)t.clock & 7) || (((uintptr_t)t.param) & (uintptr_t)(opt_size(t.param_type) - 1)) || (((uintptr_t)t.grad) & (uintptr_t)(opt_size(t.grad_type) - 1)) ||
            (!eight && (((uintptr_t)t.state0 | (uintptr_t)t.state1) & 3)))
            return fail(GSR_E_INVALID, "gsr_adamw_step: a pointer is not aligned to its type%s", "");
        ranges.add(t.param, t.n * opt_size(t.param_type), true);
        ranges.add(t.state0, t.n * (eight ? 1 : 4), true);
        ranges.add(t.state1, t.n * (eight ? 1 : 4), true);
        if (eight) ranges.add(t.window, (t.n + GSR_OPT_WINDOW - 1) / GSR_OPT_WINDOW, true);
        ranges.add(t.clock, 4 * sizeof(double), true);
        ranges.add(t.grad, t.n * opt_size(t.grad_type), false);
        ranges.add(t.lr_device, sizeof(double), false);
    }
    ranges.add(a->clip, 2 * sizeof(float), false);
    if (ranges.clash()) return fail(GSR_E_INVALID, "gsr_adamw_step: memory that the step writes overlaps other memory of the call (a tensor given twice?)%s", "");
    return GSR_OK;
}

int adamw_step(const gsr_adamw_args* a, const gsr_code_origin* origins)
{
    using namespace gsr;
    const int debug = 0;
    hipStream_t st = (hipStream_t)a->stream;
    const bool eight = a->state_bits == 8;
    int rc = adamw_check(a, origins);
    if (rc != GSR_OK || a->n_tensors == 0) return rc;
    rc = select_device_of(a->tensors[0].clock);
    if (rc != GSR_OK) return rc;
    OptArgs k;
    k.beta1 = a->beta1; k.beta2 = a->beta2;
    k.b1 = (float)a->beta1; k.b2 = (float)a->beta2; k.c1 = (float)(1.0 - a->beta1); k.c2 = (float)(1.0 - a->beta2); k.eps = (float)a->eps;
    k.clip = a->clip;
    const double span = eight ? opt_span(a->beta1, a->beta2) : 1.0;
    k.per_unit = (float)(127.0 / span);
    for (int i = 0; i < a->n_tensors; ) {
        const int count = std::min(GSR_OPT_MAX, a->n_tensors - i);
        long long bytes = 0;
        for (int j = i; j < i + count; j++) {
            const gsr_opt_tensor& t = a->tensors[j];
            bytes += t.n * (opt_size(t.param_type) + opt_size(t.grad_type) + (eight ? 2 : 8));
        }
        k.count = count;
        uint32_t groups = 0;
        for (int j = 0; j < count; j++, i++) {
            const gsr_opt_tensor& t = a->tensors[i];
            OptTensor& o = k.t[j];
            o.p = t.param; o.g = t.grad; o.s0 = t.state0; o.s1 = t.state1; o.window = t.window; o.clock = t.clock; o.lr_device = t.lr_device;
            o.lr = t.lr; o.decay = t.weight_decay; o.n = t.n; o.first = groups;
            o.unit = (float)((eight && origins ? opt_span(origins[i].beta1, origins[i].beta2) : span) / 127.0);
            o.key = a->seed * 0x9E3779B1u + ((eight && origins ? origins[i].place : (uint32_t)i) + 1u) * 0x85EBCA77u;
            const bool aligned = opt_aligned(t.param, opt_size(t.param_type)) && opt_aligned(t.grad, opt_size(t.grad_type)) &&
                                 opt_aligned(t.state0, eight ? 1 : 4) && opt_aligned(t.state1, eight ? 1 : 4);
            o.types = t.param_type | t.grad_type << 4 | (aligned ? GSR_T_ALIGNED : 0);
            groups += (uint32_t)((t.n + GSR_OPT_CHUNK - 1) / GSR_OPT_CHUNK);
        }
        const dim3 grid(std::max(1u, groups)), block(GSR_OPT_THREADS);
        const bool stream_past = opt_stream(bytes);
        if (eight && stream_past) hipLaunchKernelGGL(k_adamw8<true>, grid, block, 0, st, k);
        else if (eight) hipLaunchKernelGGL(k_adamw8<false>, grid, block, 0, st, k);
        else if (stream_past) hipLaunchKernelGGL(k_adamw<true>, grid, block, 0, st, k);
        else hipLaunchKernelGGL(k_adamw<false>, grid, block, 0, st, k);
        LAUNCHCHK(eight ? "k_adamw8" : "k_adamw");
        if (grid.x > GSR_OPT_TICKETS) {
            hipLaunchKernelGGL(k_adamw_advance, dim3(1), dim3(64), 0, st, k);
            LAUNCHCHK("k_adamw_advance");
        }
    }
    return 0;
}

int adamw_moments(int n_tensors, const gsr_moment_tensor* tensors, double beta1, double beta2, int type, void* stream)
{
    using namespace gsr;
    const int debug = 0;
    hipStream_t st = (hipStream_t)stream;
    if (n_tensors < 0 || (n_tensors > 0 && !tensors)) return fail(GSR_E_INVALID, "gsr_adamw_moments: NULL pointer%s", "");
    if (!opt_type_ok(type)) return fail(GSR_E_INVALID, "gsr_adamw_moments: unknown type%s", "");
    if (!opt_spannable(beta1, beta2)) return fail(GSR_E_INVALID, "gsr_adamw_moments: 0 <= beta1, beta1^2 < beta2 < 1 required%s", "");
    OptRanges ranges;
    const void* any = nullptr;
    for (int i = 0; i < n_tensors; i++) {
        const gsr_moment_tensor& t = tensors[i];
        if (t.n < 0 || t.n > kOptMaxElements) return fail(GSR_E_INVALID, "gsr_adamw_moments: bad tensor size%s", "");
        if (t.n > 0 && (!t.rms || !t.ratio || !t.window || !t.exp_avg_out || !t.rms_out)) return fail(GSR_E_INVALID, "gsr_adamw_moments: NULL pointer%s", "");
        if (((uintptr_t)t.exp_avg_out | (uintptr_t)t.rms_out) & (uintptr_t)(opt_size(type) - 1)) return fail(GSR_E_INVALID, "gsr_adamw_moments: a pointer is not aligned to its type%s", "");
        ranges.add(t.rms, t.n, false); ranges.add(t.ratio, t.n, false); ranges.add(t.window, (t.n + GSR_OPT_WINDOW - 1) / GSR_OPT_WINDOW, false);
        ranges.add(t.exp_avg_out, t.n * opt_size(type), true); ranges.add(t.rms_out, t.n * opt_size(type), true);
        if (t.n > 0) any = t.rms;
    }
    if (!any) return 0;
    if (ranges.clash()) return fail(GSR_E_INVALID, "gsr_adamw_moments: an output overlaps other memory of the call%s", "");
    int rc = select_device_of(any);
    if (rc != GSR_OK) return rc;
    MomentArgs k;
    k.unit = (float)(opt_span(beta1, beta2) / 127.0);
    k.type = type; k.count = 0;
    uint32_t groups = 0;
    for (int i = 0; i < n_tensors; i++) {
        const gsr_moment_tensor& t = tensors[i];
        if (t.n > 0) {
            MomentTensor& o = k.t[k.count++];
            o.rms = t.rms; o.ratio = t.ratio; o.window = t.window; o.exp_avg = t.exp_avg_out; o.root = t.rms_out; o.n = t.n; o.first = groups;
            o.aligned = opt_aligned(t.rms, 1) && opt_aligned(t.ratio, 1) && opt_aligned(t.exp_avg_out, opt_size(type)) && opt_aligned(t.rms_out, opt_size(type));
            groups += (uint32_t)((t.n + GSR_OPT_CHUNK - 1) / GSR_OPT_CHUNK);
        }
        const bool full = k.count == GSR_OPT_MAX;
        if (k.count == 0 || (!full && i + 1 < n_tensors)) continue;
        hipLaunchKernelGGL(k_moments8, dim3(groups), dim3(GSR_OPT_THREADS), 0, st, k);
        LAUNCHCHK("k_moments8");
        k.count = 0; groups = 0;
    }
    return 0;
}

int norm_launches(int n_tensors) { return (n_tensors + GSR_NORM_MAX - 1) / GSR_NORM_MAX; }

int grad_norm(int n_tensors, const void* const* grads, const long long* numels, const int* types, float max_norm, float* out,
              gsr_resize_fn workspace, void* workspace_ctx, void* stream)
{
    using namespace gsr;
    const int debug = 0;
    hipStream_t st = (hipStream_t)stream;
    if (n_tensors < 0 || (n_tensors > 0 && (!grads || !numels || !types)) || !out || !workspace) return fail(GSR_E_INVALID, "gsr_grad_norm: NULL pointer%s", "");
    if (!(max_norm >= 0.0f)) return fail(GSR_E_INVALID, "gsr_grad_norm: max_norm >= 0 required%s", "");
    for (int i = 0; i < n_tensors; i++) {
        if (numels[i] < 0 || numels[i] > kOptMaxElements) return fail(GSR_E_INVALID, "gsr_grad_norm: bad tensor size%s", "");
        if (!opt_type_ok(types[i])) return fail(GSR_E_INVALID, "gsr_grad_norm: unknown type%s", "");
        if (numels[i] > 0 && (!grads[i] || ((uintptr_t)grads[i] & (uintptr_t)(opt_size(types[i]) - 1)))) return fail(GSR_E_INVALID, "gsr_grad_norm: NULL or unaligned gradient%s", "");
    }
    int rc = select_device_of(out);
    if (rc != GSR_OK) return rc;
    double* partial = (double*)workspace(workspace_ctx, gsr_grad_norm_bytes(n_tensors));
    if (!partial) return fail(GSR_E_ALLOC, "workspace callback returned NULL%s", "");
    NormArgs k;
    k.count = 0; k.chunks = 0;
    int sums = 0;
    for (int i = 0; i < n_tensors; i++) {
        if (numels[i] > 0) {
            k.t[k.count++] = {grads[i], numels[i], k.chunks, types[i] | (opt_aligned(grads[i], opt_size(types[i])) ? GSR_T_ALIGNED : 0)};
            k.chunks += (uint32_t)((numels[i] + GSR_OPT_CHUNK - 1) / GSR_OPT_CHUNK);
        }
        const bool full = k.count == GSR_NORM_MAX;
        if (k.count == 0 || (!full && i + 1 < n_tensors)) continue;
        k.partial = partial + sums;
        // up to 32 k elements: one workgroup, one launch (a call for 16 k elements 9.7 us, in two launches 12.9)
        const bool alone = k.chunks <= 8 && sums == 0 && i + 1 == n_tensors;
        k.max_norm = max_norm; k.out = alone ? out : nullptr;
        const int grid = alone ? 1 : opt_grid(k.chunks);
        hipLaunchKernelGGL(k_grad_norm, dim3(grid), dim3(GSR_OPT_THREADS), 0, st, k);
        LAUNCHCHK("k_grad_norm");
        if (alone) return 0;
        sums += grid;
        k.count = 0; k.chunks = 0;
    }
    hipLaunchKernelGGL(k_grad_norm_finish, dim3(1), dim3(GSR_OPT_THREADS), 0, st, (const double*)partial, sums, max_norm, out);
    LAUNCHCHK("k_grad_norm_finish");
    return 0;
}

struct EvictWs { uint32_t* hist; uint32_t* found; uint2* counts; float* total; };
size_t carve_evict(char* base, int P, EvictWs& w)
{
    Carver c(base);
    w.hist = c.take<uint32_t>(3 * GSR_EV_BINS);
    w.found = c.take<uint32_t>(6);
    w.counts = c.take<uint2>(GSR_EV_TILES);
    w.total = c.take<float>(P > 0 ? (size_t)P : 1);
    return c.size();
}

int evict_rows(const gsr_evict_args* a)
{
    using namespace gsr;
    const int debug = 0;
    hipStream_t st = (hipStream_t)a->stream;
    if (a->P < 0 || a->n_views < 0 || a->n_tensors < 0) return fail(GSR_E_INVALID, "gsr_evict_rows: negative size%s", "");
    if (!(a->recent >= 0 && a->recent <= a->keep && a->keep <= a->P)) return fail(GSR_E_INVALID, "gsr_evict_rows: 0 <= recent <= keep <= P required%s", "");
    if (a->n_tensors > 0 && !a->tensors) return fail(GSR_E_INVALID, "gsr_evict_rows: NULL pointer%s", "");
    for (int i = 0; i < a->n_tensors; i++) {
        const gsr_row_tensor& t = a->tensors[i];
        if (t.row_bytes < 0 || t.row_bytes > 0x7fffffffLL || t.row_bytes > 2 * kOptMaxElements / std::max(1, a->P)) return fail(GSR_E_INVALID, "gsr_evict_rows: bad row size%s", "");
        if (a->keep > 0 && t.row_bytes > 0 && (!t.src || !t.dst || (t.src_window != nullptr) != (t.dst_window != nullptr)))
            return fail(GSR_E_INVALID, "gsr_evict_rows: NULL pointer%s", "");
    }
    if (a->keep == 0) return 0;
    if (!a->scores || !a->kept || !a->scores_out || !a->workspace || (a->n_views > 0 && !a->weights)) return fail(GSR_E_INVALID, "gsr_evict_rows: NULL pointer%s", "");
    OptRanges ranges;
    ranges.add(a->scores, 4LL * a->P, false); ranges.add(a->weights, 4LL * a->P * a->n_views, false);
    ranges.add(a->kept, 8LL * a->keep, true); ranges.add(a->scores_out, 4LL * a->keep, true);
    for (int i = 0; i < a->n_tensors; i++) {
        const gsr_row_tensor& t = a->tensors[i];
        ranges.add(t.src, t.row_bytes * a->P, false); ranges.add(t.dst, t.row_bytes * a->keep, true);
        if (t.src_window) {
            ranges.add(t.src_window, (t.row_bytes * a->P + GSR_OPT_WINDOW - 1) / GSR_OPT_WINDOW, false);
            ranges.add(t.dst_window, (t.row_bytes * a->keep + GSR_OPT_WINDOW - 1) / GSR_OPT_WINDOW, true);
        }
    }
    if (ranges.clash()) return fail(GSR_E_INVALID, "gsr_evict_rows: an output overlaps other memory of the call%s", "");
    int rc = select_device_of(a->scores);
    if (rc != GSR_OK) return rc;
    EvictWs w;
    char* ws = (char*)a->workspace(a->workspace_ctx, carve_evict(nullptr, a->P, w));
    if (!ws) return fail(GSR_E_ALLOC, "workspace callback returned NULL%s", "");
    carve_evict(ws, a->P, w);
    EvictArgs e;
    e.P = a->P; e.views = a->n_views; e.old = a->P - a->recent; e.k = a->keep - a->recent; e.decay = a->decay;
    e.scores = a->scores; e.weights = a->weights; e.total = w.total; e.hist = w.hist; e.found = w.found; e.counts = w.counts;
    e.kept = a->kept; e.scores_out = a->scores_out;
    if (a->P <= GSR_EV_SMALL) {          // one workgroup, one launch
        hipLaunchKernelGGL(k_evict_small, dim3(1), dim3(1024), 0, st, e);
        LAUNCHCHK("k_evict_small");
    } else {
        const long long tiles = std::min<long long>(((long long)a->P + GSR_EV_TILE - 1) / GSR_EV_TILE, GSR_EV_TILES), per = ((long long)a->P + tiles - 1) / tiles;
        e.tile_rows = (int)((per + GSR_EV_TILE - 1) / GSR_EV_TILE * GSR_EV_TILE);
        const int n_tiles = (int)(((long long)a->P + e.tile_rows - 1) / e.tile_rows);
        if (e.k > 0 && e.k < e.old) {
            ClearRanges cr = {};
            cr.p[0] = w.hist; cr.n[0] = 3 * GSR_EV_BINS;
            hipLaunchKernelGGL(k_refine_init, dim3(3 * GSR_EV_BINS / GSR_BLOCK), dim3(GSR_BLOCK), 0, st, cr, PoseLoadArgs{});
            LAUNCHCHK("k_refine_init");
        }
        hipLaunchKernelGGL(k_evict_scores, dim3((unsigned)std::min<long long>(((long long)a->P + 2047) / 2048, 256)), dim3(512), 0, st, e);
        LAUNCHCHK("k_evict_scores");
        if (e.k > 0 && e.k < e.old) {
            const dim3 blocks((unsigned)std::min<long long>(((long long)a->P + 8191) / 8192, 256));
            hipLaunchKernelGGL(k_evict_hist<2>, blocks, dim3(1024), 0, st, e);
            LAUNCHCHK("k_evict_hist<2>");
            hipLaunchKernelGGL(k_evict_hist<3>, blocks, dim3(1024), 0, st, e);
            LAUNCHCHK("k_evict_hist<3>");
        }
        hipLaunchKernelGGL(k_evict_count, dim3(n_tiles), dim3(256), 0, st, e);
        LAUNCHCHK("k_evict_count");
        hipLaunchKernelGGL(k_evict_emit, dim3(n_tiles), dim3(256), 0, st, e);
        LAUNCHCHK("k_evict_emit");
    }
    RowArgs k;
    k.keep = a->keep; k.kept = a->kept; k.count = 0;
    uint32_t groups = 0;
    for (int i = 0; i < a->n_tensors; i++) {
        const gsr_row_tensor& t = a->tensors[i];
        if (t.row_bytes > 0) {
            RowTensor& o = k.t[k.count++];
            const uintptr_t bits = (uintptr_t)t.src | (uintptr_t)t.dst | (uintptr_t)t.row_bytes;
            o.src = t.src; o.dst = t.dst; o.src_window = t.src_window; o.dst_window = t.dst_window; o.first = groups;
            o.unit = t.src_window ? 1 : (bits & 15) == 0 ? 16 : (bits & 7) == 0 ? 8 : (bits & 3) == 0 ? 4 : (bits & 1) == 0 ? 2 : 1;
            o.row = t.row_bytes / o.unit;
            o.large = t.row_bytes * a->P >= (1LL << 32);
            // y ceil(2^32 / row) exceeds y 2^32 / row by less than y: the quotient is right while y row < 2^32
            o.magic = o.row > 1 && (o.row + GSR_EV_CHUNK) * o.row < (1LL << 32) ? (uint32_t)(((1LL << 32) + o.row - 1) / o.row) : 0u;
            const long long chunk = o.unit == 1 ? GSR_EV_CHUNK : GSR_OPT_CHUNK;
            groups += (uint32_t)((o.row * a->keep + chunk - 1) / chunk);
        }
        const bool full = k.count == GSR_OPT_MAX || groups > 1u << 22;
        if (k.count == 0 || (!full && i + 1 < a->n_tensors)) continue;
        hipLaunchKernelGGL(k_evict_rows, dim3(groups), dim3(GSR_OPT_THREADS), 0, st, k);
        LAUNCHCHK("k_evict_rows");
        k.count = 0; groups = 0;
    }
    return 0;
}

// std::vector and std::sort may throw; nothing may leave a C entry point that way.
template <class F>
int no_throw(F f)
{
    try { return f(); }
    catch (const std::exception& e) { return fail(GSR_E_ALLOC, "host memory: %s", e.what()); }
    catch (...) { return fail(GSR_E_ALLOC, "host exception%s", ""); }
}
}  // namespace
