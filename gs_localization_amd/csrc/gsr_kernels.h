// gsr_kernels.h -- gfx950 kernels of the splat rasterizer hot path (forward + backward).
// Included once by gsr_api.hip.  Per-kernel roofline notes are in DESIGN.md section "Kernels".
#pragma once
#include "gsr_device.h"

namespace gsr {

// Diagnostic builds (GSR_TIMING=1 python gs_localization_amd/build.py): per-phase shader-clock totals of the two
// compositing kernels, summed over waves (lane 0 of each wave keeps the running totals in scalar registers and
// flushes them once at the end).  Read back with gsr_debug_timing(); slots 0-15 = K6, 16-31 = K7.
#ifndef GSR_TIMING
#define GSR_TIMING 0
#endif
#if GSR_TIMING
#define GSR_TIM_WAVES (16384 * 4)
__device__ unsigned long long g_tim[4][GSR_TIM_WAVES][12];      // [kernel][wave][slot]: every wave owns its row, no atomics
// ... and, of the LAST launch only (overwritten, not added): the wave's first and last instant on the 100 MHz wall clock -- a timeline of
// one launch's workgroups (tools/dbg/timeline.py: is a kernel's duration its throughput or the tail of one chain?)
__device__ unsigned long long g_tim_span[4][GSR_TIM_WAVES][2];
__device__ unsigned long long g_tim_last[4][GSR_TIM_WAVES][12];      // ... and its phase slots
#define GSR_T_DECL long long t_prev_ = clock64(); const long long t_start_ = t_prev_; long long t_acc_[12] = {0,0,0,0,0,0,0,0,0,0,0,0}; const unsigned long long t_wall0_ = wall_clock64();
#define GSR_T_TICK(slot) { const long long now_ = clock64(); t_acc_[slot] += now_ - t_prev_; t_prev_ = now_; }
#define GSR_T_COUNT(slot, v) { t_acc_[slot] += (v); }
// -DGSR_TIMING_ORDER: slots 4 / 6 / 7 of k_render_fwd show the lazy ordering's sub-phases (sample + threshold search, gather pass, sort)
// instead; what they usually hold is added to slot 5
#define GSR_T_PARAMS , long long& t_prev_, long long (&t_acc_)[12]
#define GSR_T_ARGS , t_prev_, t_acc_
#ifdef GSR_TIMING_ORDER
#define GSR_TO(slot) 5
#define GSR_T_TICK_O(slot) GSR_T_TICK(slot)
#else
#define GSR_TO(slot) slot
#define GSR_T_TICK_O(slot)
#endif
#define GSR_T_FLUSH(base) t_acc_[9] = clock64() - t_start_; if ((threadIdx.x & 63) == 0 && blockIdx.x * 4 + (threadIdx.x >> 6) < GSR_TIM_WAVES) { for (int q_ = 0; q_ < 12; q_++) { g_tim[(base) / 16][blockIdx.x * 4 + (threadIdx.x >> 6)][q_] += (unsigned long long)t_acc_[q_]; g_tim_last[(base) / 16][blockIdx.x * 4 + (threadIdx.x >> 6)][q_] = (unsigned long long)t_acc_[q_]; } g_tim_span[(base) / 16][blockIdx.x * 4 + (threadIdx.x >> 6)][0] = t_wall0_; g_tim_span[(base) / 16][blockIdx.x * 4 + (threadIdx.x >> 6)][1] = wall_clock64(); }
// (workgroups of `wpb` waves)
#define GSR_T_FLUSH_W(base, wpb) t_acc_[9] = clock64() - t_start_; if ((threadIdx.x & 63) == 0 && blockIdx.x * (wpb) + (threadIdx.x >> 6) < GSR_TIM_WAVES) { for (int q_ = 0; q_ < 12; q_++) { g_tim[(base) / 16][blockIdx.x * (wpb) + (threadIdx.x >> 6)][q_] += (unsigned long long)t_acc_[q_]; g_tim_last[(base) / 16][blockIdx.x * (wpb) + (threadIdx.x >> 6)][q_] = (unsigned long long)t_acc_[q_]; } g_tim_span[(base) / 16][blockIdx.x * (wpb) + (threadIdx.x >> 6)][0] = t_wall0_; g_tim_span[(base) / 16][blockIdx.x * (wpb) + (threadIdx.x >> 6)][1] = wall_clock64(); }
#else
#define GSR_T_DECL
#define GSR_T_TICK(slot)
#define GSR_T_COUNT(slot, v)
#define GSR_T_FLUSH(base)
#define GSR_T_FLUSH_W(base, wpb)
#define GSR_T_TICK_O(slot)
#define GSR_TO(slot) slot
#define GSR_T_PARAMS
#define GSR_T_ARGS
#endif

// Device-side guards of the native refinement loop (gsr_refine).  The host enqueues kernel GROUPS (preprocess, compositing,
// backward compositing, chain rule + pose step) one ahead of the statuses it has seen, so every kernel of a group checks
// two device words itself:
//   poison : (tag << 2) | flags of the last group whose speculative forward failed its verification (flag bit 0: a tile ran out
//            of list with an unsaturated pixel; bit 1: a bin overflowed).  A kernel is poisoned iff the word carries ITS OWN
//            group's tag: the rest of that group (loss, backward, pose step) is skipped, the pose does not move -- and the NEXT
//            group, already enqueued, runs as the retry of the same iteration without any host intervention: it bins with the
//            bounds the failed forward recorded, in which every failed tile has no bound (complete list) and every other tile
//            the exact depth it needed at this very pose.  Tags only grow, so nothing ever has to be cleared.
//   conv   != 0 : the pose update already converged; loss, backward and pose step are skipped (frozen).
// Both pointers are NULL outside the native loop.
struct LoopGuard {
    const uint32_t* poison; const float* conv; uint32_t tag;
    __device__ __forceinline__ bool poisoned() const { return poison != nullptr && (*poison >> 2) == tag; }
    __device__ __forceinline__ bool frozen() const { return poisoned() || (conv != nullptr && *conv != 0.f); }
};
#ifndef GSR_HOLD_FORWARDS
#define GSR_HOLD_FORWARDS 32u    // forwards a tile goes without a depth bound after failing a verification (native loop)
#endif
#define GSR_FAIL_BOUND 1u        // poison / fail word flags
#define GSR_FAIL_OVERFLOW 2u

// ---------------------------------------------------------------------------------------------
// K1  per-Gaussian preprocess (replaces forward.cu:155-256 preprocessCUDA).
// One lane per Gaussian; HBM-streaming: reads 44+12M B, writes <= 80 B per Gaussian.
// ---------------------------------------------------------------------------------------------
// ---------------------------------------------------------------------------------------------
// Exact tile culling.  The reference emits one instance for every tile of the bounding SQUARE of
// radius ceil(3 sigma_max) (forward.cu:229-237).  An instance can only change a pixel if
// alpha = o*exp(-q) >= 1/255 there (forward.cu:346-348), i.e. q <= ln(255 o).  For each tile of the
// reference rectangle we compute the exact minimum of the convex quadratic q over the tile's pixel
// rectangle and drop the instance when even that minimum (minus a safety slack covering fp32
// rounding of q in the compositing kernels) is above the threshold: a dropped instance would have
// been skipped by every pixel of the tile, so images and gradients are unchanged while the binned
// list gets shorter.  Never ADDS tiles outside the reference rectangle; `radii` is still the
// reference's value.
// ---------------------------------------------------------------------------------------------
struct TileTest {
    float mx, my, A, B, C, det, twoq, dxe, dye, invA, dyext;
    bool cull;       // false: conic not positive definite -> keep every tile of the rectangle
    bool none;       // opacity so low that alpha < 1/255 everywhere
};
__device__ __forceinline__ TileTest make_tile_test(float2 m, float3 conic, float opacity)
{
    TileTest t;
    t.mx = m.x; t.my = m.y; t.A = conic.x; t.B = conic.y; t.C = conic.z;
    t.det = conic.x * conic.z - conic.y * conic.y;
    t.cull = (conic.x > 0.f) && (conic.z > 0.f) && (t.det > 0.f);
#ifdef GSR_NO_CULL      // diagnostic build (tools/cull_check.py): every tile of the reference rectangle, every quadrant
    t.cull = false;
#endif
    // q <= ln(255 o) + slack.  The slack (0.02 in q, i.e. 2 % in alpha) covers the fp32 rounding of q in
    // the compositing kernels, also for strongly correlated conics where q is a difference of large terms.
    const float qmax = (opacity > 0.f) ? (__logf(255.f * opacity) + 0.02f) : -1.f;
    t.none = t.cull && (qmax < 0.f);
    t.twoq = 2.f * fmaxf(qmax, 0.f);
    // extreme points of the ellipse q = qmax (d = mean - pixel): dx = +-dxe at dy = -+B dxe / C, and |dy| <= dyext
    // (hardware rcp / sqrt, ~1 ulp: the spans are widened by 0.01 px, exact rounding is not needed here)
    const float rdet = t.cull ? __builtin_amdgcn_rcpf(t.det) : 0.f;
    t.invA = t.cull ? __builtin_amdgcn_rcpf(t.A) : 0.f;
    t.dxe = t.cull ? __builtin_amdgcn_sqrtf(t.twoq * t.C * rdet) : 0.f;
    t.dye = t.cull ? (-t.B * t.dxe * __builtin_amdgcn_rcpf(t.C)) : 0.f;
    t.dyext = t.cull ? __builtin_amdgcn_sqrtf(t.twoq * t.A * rdet) : 0.f;
    return t;
}
// Shrinks the reference's tile rectangle [x0, x1) x [y0, y1) to the tiles the bounding box of the ellipse q <= qmax reaches
// (the rows and columns cut off have empty spans); widened by 0.01 px like the spans.  May come out empty.
__device__ __forceinline__ void clip_rect(const TileTest& t, int& x0, int& y0, int& x1, int& y1)
{
    if (!t.cull) return;
    if (t.none) { x1 = x0; y1 = y0; return; }
    const float ex = t.dxe * 1.0001f + 0.01f, ey = t.dyext * 1.0001f + 0.01f;      // pixels mx - ex ... mx + ex, my - ey ... my + ey
    x0 = max(x0, (int)ceilf((t.mx - ex - (float)(GSR_TILE - 1)) * (1.f / GSR_TILE)));
    x1 = max(x0, min(x1, (int)floorf((t.mx + ex) * (1.f / GSR_TILE)) + 1));
    y0 = max(y0, (int)ceilf((t.my - ey - (float)(GSR_TILE - 1)) * (1.f / GSR_TILE)));
    y1 = max(y0, min(y1, (int)floorf((t.my + ey) * (1.f / GSR_TILE)) + 1));
}
// Tiles [lo, hi] (inclusive, within [x0, x1)) of tile row ty that the ellipse q <= qmax can reach; empty if lo > hi.
// For a fixed dy the ellipse spans dx in [(-B dy - s) / A, (-B dy + s) / A] with s = sqrt(A twoq - det dy^2).  The upper end
// is a concave function of dy that peaks at the ellipse's +x extreme point (dy = dye), the lower end a convex one with its
// minimum at the -x extreme point (dy = -dye): over the row's band of pixel rows each is extremal at that dy clamped into
// the band -- one evaluation (one sqrt) per end, no case distinction.  Exact; widened by 0.01 px.
__device__ __forceinline__ void row_span(const TileTest& t, int ty, int x0, int x1, int& lo, int& hi)
{
    if (!t.cull) { lo = x0; hi = x1 - 1; return; }
    lo = 1; hi = 0;
    if (t.none) return;
    const float dyh = t.my - (float)(ty * GSR_TILE), dyl = dyh - (float)(GSR_TILE - 1);   // d = mean - pixel
    const float dy1 = fminf(dyh, fmaxf(dyl, t.dye)), dy2 = fminf(dyh, fmaxf(dyl, -t.dye));
    const float at = t.A * t.twoq;
    const float disc1 = at - t.det * dy1 * dy1, disc2 = at - t.det * dy2 * dy2;
    // (a clamped dy lies outside the ellipse's y-extent only if the whole band does; a hair of negative rounding is let through)
    if (fminf(disc1, disc2) < -1e-3f * at) return;
    const float dmax = (__builtin_amdgcn_sqrtf(fmaxf(disc1, 0.f)) - t.B * dy1) * t.invA;
    const float dmin = (-__builtin_amdgcn_sqrtf(fmaxf(disc2, 0.f)) - t.B * dy2) * t.invA;
    const float pa = t.mx - dmax - 0.01f, pb = t.mx - dmin + 0.01f;        // pixel x-interval
    lo = max(x0, (int)ceilf((pa - (float)(GSR_TILE - 1)) * (1.f / GSR_TILE)));
    hi = min(x1 - 1, (int)floorf(pb * (1.f / GSR_TILE)));
}

// ---------------------------------------------------------------------------------------------
// Bin-by-tile path of the native loop.  Once the speculative depth bounds have cut the per-tile lists down to
// a few hundred entries, neither global sort is needed: k_preprocess appends (depth bits << 32 | index) straight
// into fixed-capacity per-tile bins (one returning atomic on the tile's cursor per instance), and the compositing
// kernel sorts each tile's bin in LDS -- by (depth bits, index), the same total order as the reference's stable
// radix sort of (tile | depth) keys (rasterizer_impl.cu:304-309).  No prefix sum, no host read of the instance
// count.  A tile with more than GSR_LSORT_CAP entries reports failure and the host redoes the forward on the
// global-sort path.
// ---------------------------------------------------------------------------------------------
#define GSR_LSORT_CAP 2048        // bin capacity = longest list the in-LDS sort takes
// Bins (and the sorted index lists next to them) sit capacity + GSR_BIN_PAD entries apart: capacities are powers of two, and a
// thousand tiles whose bins all START at multiples of 64 KB put every workgroup's first reads and the preprocess's appends on the
// same few memory channels (measured with complete lists, 2 800 keys per tile: compositing 79 us against 62 with the keys packed
// back to back).  160 entries = 1 280 B of keys / 640 B of indices: an odd number of 256-byte granules per tile.
#define GSR_BIN_PAD 160
#define GSR_CURSOR_STRIDE 16      // cursors sit 64 B apart: the atomics of neighbouring tiles go to different lines
#ifndef GSR_COOP_AREA
#define GSR_COOP_AREA 8           // rectangles with more tiles than this are walked by the whole wave
#endif

// ---------------------------------------------------------------------------------------------
// Work lists.  After the preprocess only the Gaussians that were binned into at least one tile ("survivors": a few
// per cent of the map in a speculative iteration of the native loop, the visible ones otherwise) have any work left in
// the forward (SH colour) and in the per-Gaussian half of the backward (chain rule).  k_preprocess appends them to
// GSR_SURV_LISTS sub-lists -- workgroup b to sub-list b mod GSR_SURV_LISTS, one wave-aggregated returning atomic per wave
// that has any; a single counter would serialise thousands of same-address atomics at the memory side (tens of ns each) --
// and k_sh_color / k_preprocess_bwd walk the lists on dense lanes instead of scanning all P Gaussians for the few that
// matter (48 MB of accumulator records + 4 MB of flags per iteration at 1 M Gaussians).  Sub-list s owns ids[s * cap ...),
// cap = the number of Gaussians its workgroups cover; the counters sit 256 B apart.  Order inside a list is arrival order:
// every consumer writes per-Gaussian rows or adds into sums, neither depends on it.
// ---------------------------------------------------------------------------------------------
#define GSR_SURV_LISTS 64
#define GSR_SURV_CSTRIDE 64
#ifndef GSR_LEAN_PER_LANE
#define GSR_LEAN_PER_LANE 4      // Gaussians per lane of k_preprocess_lean
static_assert(GSR_LEAN_PER_LANE == 4 && GSR_LEAN_PER_LANE * 256 == 1024, "surv_cap() and k_preprocess_bin's virtual blocks (idx >> 10) assume 1 024-Gaussian stretches: change them together");
#endif
#ifndef GSR_LEAN_WINDOW
#define GSR_LEAN_WINDOW 256      // (64: 58 / 128 us on the sorted S-1M-640 / S-3M-cam; 256: 45 / 68; 1 024: 43 / 68; random order: 35 / 60 whichever)
#endif
// ^ waves that share their Gaussians segment by segment (k_preprocess_lean); the grid is a multiple of a quarter of it
#ifndef GSR_LEAN_POOL
#define GSR_LEAN_POOL 1          // waves of a workgroup that pool their candidates for one exact pass (1, 2 or 4)
#endif
struct SurvLists { uint32_t* ids; uint32_t* n; uint32_t cap; };
static inline uint32_t surv_cap(int P)
{
    // (what the workgroups b = s mod GSR_SURV_LISTS of k_preprocess / k_preprocess_lean cover: 256 / GSR_LEAN_PER_LANE x 256 Gaussians
    // each; k_preprocess_bin's 2 048-Gaussian workgroups file their survivors by 1 024-Gaussian stretch, idx >> 10.  The largest of these
    // sizes the sub-lists and bounds the others: ceil(n / 64) x 256 <= ceil(n / 256) x 1 024.)
    const uint32_t per = GSR_LEAN_PER_LANE * GSR_BLOCK;
    const uint32_t blocks = ((uint32_t)(P > 0 ? P : 1) + per - 1) / per;
    return (blocks + GSR_SURV_LISTS - 1) / GSR_SURV_LISTS * per;
}
// workgroups (of one wave) a list consumer is launched with: a multiple of GSR_SURV_LISTS, at most `resident`
static inline int surv_grid(int P, int resident)
{
    const int chunks = (int)((surv_cap(P) + 63u) / 64u);                     // longest possible sub-list, in 64-entry chunks
    const int per_list = chunks < resident / GSR_SURV_LISTS ? chunks : resident / GSR_SURV_LISTS;
    return GSR_SURV_LISTS * (per_list > 0 ? per_list : 1);
}

// The per-Gaussian gradient rows (native loop: maintained from one iteration to the next through the dirty bits, see
// PreBwdArgs::dirty).  bit 0 of a dirty byte = the small rows hold values, bit 1 = the dL_dsh row does.
struct GradRows {
    float* mean2D; float* conic; float* opacity; float* color; float* mean3D; float* cov3D; float* sh; float* scale; float* rot; int M;
};
__device__ __forceinline__ void zero_grad_rows(const GradRows& r, size_t idx, bool small, bool sh_row)
{
    if (small) {
        r.color[3 * idx] = 0.f; r.color[3 * idx + 1] = 0.f; r.color[3 * idx + 2] = 0.f;
        r.mean2D[3 * idx] = 0.f; r.mean2D[3 * idx + 1] = 0.f;
        reinterpret_cast<float4*>(r.conic)[idx] = make_float4(0.f, 0.f, 0.f, 0.f);
        r.opacity[idx] = 0.f;
        if (r.mean3D) { r.mean3D[3 * idx] = 0.f; r.mean3D[3 * idx + 1] = 0.f; r.mean3D[3 * idx + 2] = 0.f; }
        if (r.cov3D) {
#pragma unroll
            for (int i = 0; i < 6; i++) r.cov3D[6 * idx + i] = 0.f;
        }
        if (r.scale) { r.scale[3 * idx] = 0.f; r.scale[3 * idx + 1] = 0.f; r.scale[3 * idx + 2] = 0.f; }
        if (r.rot) reinterpret_cast<float4*>(r.rot)[idx] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
    if (sh_row && r.sh)
        for (int i = 0; i < r.M * 3; i++) r.sh[idx * r.M * 3 + i] = 0.f;
}

// Packed per-Gaussian splat record (GSR_REC_STRIDE floats = 48 B): the forward's whole per-Gaussian screen-space state,
//   0 x  1 y  2 B2  3 C2 | 4 A2  5 opacity  6 depth  7 - | 8 r  9 g  10 b  11 -
// with the conic (a, b, c) stored pre-multiplied for the exponent, A2 = -a/2 log2e, B2 = -b log2e, C2 = -c/2 log2e (see
// k_render_fwd).  Written by k_preprocess (two 16-B stores; the colour too when it is precomputed) and k_sh_color (one);
// gathered by the compositing kernels' staging, the exact-bin walks and the chain-rule kernel with 16-B loads of one
// contiguous record (round 1 kept xy / conic / colour / depth in four arrays: four cache lines per gathered splat), and
// read by K7's walk with SCALAR loads: a list entry is the same for all 64 lanes of a wave, so its record belongs in scalar
// registers -- 48 B per wave through the scalar cache instead of 40 B x 64 lanes through the LDS pipe, which K7 kept 65 % busy
// with exactly that.  Record P is the null splat (all zero).
#define GSR_REC_STRIDE 12
#define GSR_LOG2E 1.4426950408889634f
#define GSR_CONST_AS __attribute__((address_space(4)))
typedef float gsr_sf8 __attribute__((ext_vector_type(8)));
typedef float gsr_sf4 __attribute__((ext_vector_type(4)));
struct SplatRec { float x, y, a, b, c, opacity, depth; };      // (a, b, c: the conic as stored, recovered from A2, B2, C2 to 1 ulp)
__device__ __forceinline__ SplatRec load_splat_rec(const float* __restrict__ rec, uint32_t id)
{
    const float4* r = reinterpret_cast<const float4*>(rec + (size_t)id * GSR_REC_STRIDE);
    const float4 r0 = r[0], r1 = r[1];
    SplatRec o;
    o.x = r0.x; o.y = r0.y; o.b = r0.z * (-1.0f / GSR_LOG2E); o.c = r0.w * (-2.0f / GSR_LOG2E); o.a = r1.x * (-2.0f / GSR_LOG2E);
    o.opacity = r1.y; o.depth = r1.z;
    return o;
}

struct PreArgs {
    int P, D, M, W, H, gx, gy;
    uint32_t* tile_count; int ntiles;      // exact-bin path: ntiles counter words (all copies) zeroed here for k_tile_count (nullable)
    const float* zb;                       // speculative per-tile depth bounds of the native loop (nullable): the depth each
    float zb_mul, zb_add;                  // tile had to look at; an instance is kept if z <= zb * zb_mul + zb_add
    const float* zbc; int sbx, sby;        // the same per 4x4-tile superblock (max of its tiles): quick reject; sbx x sby superblocks
    int zbc_lds;                           // k_preprocess: number of bounds staged in LDS (0: read the superblock bounds from global)
    int pyr_tiles;                         // ... 1: they are the per-TILE bounds zb (gx x gy, round 5), 0: the per-superblock bounds zbc (sbx x sby)
    int lean;                              // k_preprocess: radii of this forward are not an output (see the kernel)
    // bin-by-tile path (nullable): per-tile append cursors and fixed-capacity bins of (depth bits << 32 | index)
    uint32_t* tile_cursor; unsigned long long* bins; int bin_cap;      // (bin_cap: entries per bin; bins sit bin_cap + GSR_BIN_PAD entries apart)
    int* n_touched;          // nullable: cleared here (one 4-B store per Gaussian) instead of by a separate memset
    LoopGuard guard;
    const float* means; const float* scales; float mod; const float* rots; const float* opac;
    const float* shs; const float* cov3D_pre; const float* colors_pre;
    const float* view; const float* proj; const float* campos;
    float tanx, tany, fx, fy;
    int* radii; float* cov3D;
    float* lam;              // [P] float4 (x, y, z, e): the mean and e = an upper bound on sqrt(lambda_max(Sigma_3D)) of every Gaussian
                             // (scale_modifier included), written next to cov3D by a cov_all forward: ALL that k_preprocess_lean's
                             // conservative test reads per Gaussian, as one 16-byte load (nullable elsewhere)
    float* rec;              // packed splat records (GSR_REC_*), P + 1 of them
    uint8_t* clamped; uint32_t* tiles_touched; ushort4* rects;
    int cov_all;             // k_preprocess: compute and store cov3D for every Gaussian, culled or not (see there)
    int sh_here;             // k_preprocess_lean: evaluate the survivors' SH colour itself (no k_sh_color launch behind it)
    int lazy_sh;             // complete lists: no k_sh_color either -- k_render_fwd evaluates the colours of the splats it stages (LazySH)
    SurvLists surv;          // work lists: k_preprocess appends, k_sh_color walks (ids nullable: no lists kept)
    // Native loop only (dirty nullable): a Gaussian that is NOT a survivor of this forward gets no gradient this iteration;
    // whatever the previous iteration left in its rows is cleared here, by the one kernel that visits every Gaussian anyway
    // (k_preprocess_bwd only sees the survivors).  Skipped on a frozen (converged) iteration, whose backward does not run.
    uint8_t* dirty; GradRows rows;
    // Native loop only (tile_order nullable): workgroup 0 turns the per-tile work the previous backward measured into this
    // iteration's launch order of the compositing kernels (see tile_order_from_work)
    // ([0]: k_render_fwd's order from the work it measured, [1]: k_render_bwd_mfma's)
    const uint32_t* tile_work[2]; uint32_t* tile_order[2]; int order_tiles;
};

// Real spherical-harmonics basis of the 3DGS convention (signs and constants as forward.cu:20-71 / sh_utils.py), degree <= 3:
// B[k](d) for the unit direction d = (x, y, z); entries above the active degree are left untouched.
__device__ __forceinline__ void sh_basis(int deg, float x, float y, float z, float* B)
{
    B[0] = kSH_C0;
    if (deg < 1) return;
    B[1] = -kSH_C1 * y; B[2] = kSH_C1 * z; B[3] = -kSH_C1 * x;
    if (deg < 2) return;
    const float xx = x * x, yy = y * y, zz = z * z, xy = x * y, yz = y * z, xz = x * z;
    B[4] = kSH_C2[0] * xy; B[5] = kSH_C2[1] * yz; B[6] = kSH_C2[2] * (2.0f * zz - xx - yy); B[7] = kSH_C2[3] * xz; B[8] = kSH_C2[4] * (xx - yy);
    if (deg < 3) return;
    B[9] = kSH_C3[0] * y * (3.0f * xx - yy); B[10] = kSH_C3[1] * xy * z; B[11] = kSH_C3[2] * y * (4.0f * zz - xx - yy);
    B[12] = kSH_C3[3] * z * (2.0f * zz - 3.0f * xx - 3.0f * yy); B[13] = kSH_C3[4] * x * (4.0f * zz - xx - yy);
    B[14] = kSH_C3[5] * z * (xx - yy); B[15] = kSH_C3[6] * x * (xx - 3.0f * yy);
}
// View-dependent colour of one Gaussian: max(0, sum_k B_k(d) sh[k] + 0.5) per channel, d the unit vector from the camera
// centre to the mean; clamp_bits records which channels were cut at zero (their gradient is masked in the backward pass).
__device__ __forceinline__ float3 sh_to_rgb(int deg, int M, float3 pos, const float* campos, const float* sh,
                                            uint8_t& clamp_bits)
{
    (void)M;
    const float vx = pos.x - campos[0], vy = pos.y - campos[1], vz = pos.z - campos[2];
    const float len = sqrtf(vx * vx + vy * vy + vz * vz);
    float B[16];
    sh_basis(deg, vx / len, vy / len, vz / len, B);
    const int nk = (deg + 1) * (deg + 1);
    float c0 = 0.f, c1 = 0.f, c2 = 0.f;
#pragma unroll
    for (int k = 0; k < 16; k++)
        if (k < nk) { c0 += B[k] * sh[k * 3]; c1 += B[k] * sh[k * 3 + 1]; c2 += B[k] * sh[k * 3 + 2]; }
    c0 += 0.5f; c1 += 0.5f; c2 += 0.5f;
    clamp_bits = (uint8_t)((c0 < 0 ? 1 : 0) | (c1 < 0 ? 2 : 0) | (c2 < 0 ? 4 : 0));
    return make_float3(fmaxf(c0, 0.0f), fmaxf(c1, 0.0f), fmaxf(c2, 0.0f));
}

// SH rows of one block staged through LDS: the 256 x M x 3 floats of a block are contiguous in HBM, so
// the block reads (writes) them as one coalesced 16-B-per-lane stream and each lane then works on its own
// row out of LDS.  Row stride 13 float4 (208 B) keeps the per-lane ds_read_b128 conflict-free.
#define GSR_SH16_ROW4 12      // float4 per 16-coefficient row
#define GSR_SH16_LDS4 13      // padded row stride in float4

// the vector path needs 16-coefficient rows and a 16-B aligned table (torch allocations always are)
__device__ __forceinline__ bool sh16_vector_ok(int M, const float* shs)
{
    return M == 16 && ((reinterpret_cast<uintptr_t>(shs) & 15u) == 0);
}
// sh_to_rgb for a lane that reads its own 16-coefficient row from global memory (the lean preprocess, lazy colours in the
// compositing kernel): the 192 B arrive as 16-B loads, six at a time, and are consumed in coefficient order (same sums as
// sh_to_rgb); half a row in flight keeps the register footprint of the callers' hot loops intact.
__device__ __forceinline__ float3 sh_row16_to_rgb(int deg, float3 pos, const float* campos, const float4* __restrict__ row4, uint8_t& clamp_bits)
{
    const float vx = pos.x - campos[0], vy = pos.y - campos[1], vz = pos.z - campos[2];
    const float len = sqrtf(vx * vx + vy * vy + vz * vz);
    float B[16];
    sh_basis(deg, vx / len, vy / len, vz / len, B);
    const int nk = (deg + 1) * (deg + 1);
    float c[3] = {0.f, 0.f, 0.f};
#pragma unroll
    for (int half = 0; half < 2; half++) {
        float4 v[6];
#pragma unroll
        for (int i = 0; i < 6; i++) v[i] = row4[6 * half + i];
#pragma unroll
        for (int i = 0; i < 6; i++) {
            const float e[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const int idx = 4 * (6 * half + i) + j, k = idx / 3, ch = idx - 3 * k;
                if (k < nk) c[ch] += B[k] * e[j];
            }
        }
        __builtin_amdgcn_sched_barrier(0);
    }
    c[0] += 0.5f; c[1] += 0.5f; c[2] += 0.5f;
    clamp_bits = (uint8_t)((c[0] < 0 ? 1 : 0) | (c[1] < 0 ? 2 : 0) | (c[2] < 0 ? 4 : 0));
    return make_float3(fmaxf(c[0], 0.0f), fmaxf(c[1], 0.0f), fmaxf(c[2], 0.0f));
}

// ---------------------------------------------------------------------------------------------
// Work-balanced launch order of the compositing kernels (native loop).  All tiles of a 640x480 image are resident at once
// (1200 workgroups on 256 CUs x 5), so K6 / K7 last as long as their slowest CU, and a tile's list is anything between a
// third and three times the mean.  Workgroups are handed to the CUs breadth-first -- blocks b, b + 256, b + 512, ... share a
// CU (tools/micro/dispatch_order.hip) -- so if the blocks are numbered by DEcreasing work, in a snake over the CUs (ranks
// 0..255 left to right, 256..511 right to left, ...), every CU gets one tile of each weight class and the heaviest tiles
// get the lightest company.  The work of a tile is what K7 measured one iteration earlier (the longest of its four waves'
// walks); the pose moves by a fraction of a pixel per iteration, so the estimate is good, and ANY permutation is correct.
// One workgroup, counting sort (the work is a small integer: groups of eight list entries, clamped to 255): histogram in LDS,
// prefix sum over the 256 classes, one returning LDS atomic per tile for its place among its equals (arrival order: any
// permutation is correct) -- three barriers, about a microsecond.  (With more tiles than resident workgroups the order is heaviest-first: the classic list-scheduling rule.)
// ---------------------------------------------------------------------------------------------
#define GSR_ORDER_MAX_TILES 65536
// (cls_of(t): the weight class of tile t, 0 ... 255, 255 = heaviest)
template <class ClsOf>
__device__ __forceinline__ void tile_order_from(ClsOf&& cls_of, uint32_t* __restrict__ order, int ntiles, uint32_t* s_cls /*[256]*/)
{
    // (the first GSR_BLOCK threads of the workgroup do the work; a wider workgroup's other threads only keep the barriers company)
    __shared__ uint32_t s_wsum[4];
    const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
    const bool act = tid < GSR_BLOCK;
    if (act) s_cls[tid] = 0u;
    __syncthreads();
    for (int t = tid; act && t < ntiles; t += GSR_BLOCK) atomicAdd(&s_cls[255u - min((uint32_t)cls_of(t), 255u)], 1u);      // slot 0 = heaviest
    __syncthreads();
    const uint32_t mine = act ? s_cls[tid] : 0u;
    uint32_t incl = mine;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const uint32_t o = __shfl_up(incl, off, 64);
        if (lane >= off) incl += o;
    }
    if (act && lane == 63) s_wsum[wv] = incl;
    __syncthreads();
    uint32_t start = incl - mine;
    for (int w = 0; act && w < wv; w++) start += s_wsum[w];
    if (act) s_cls[tid] = start;                                        // first rank of class tid
    __syncthreads();
    for (int t = tid; act && t < ntiles; t += GSR_BLOCK) {
        const int r = (int)atomicAdd(&s_cls[255u - min((uint32_t)cls_of(t), 255u)], 1u);          // rank, heaviest first
        // rank r goes to block (r / 256) * 256 + snake(r % 256)
        const int row = r >> 8, i = r & 255;
        const int in_row = min(256, ntiles - (row << 8));
        order[(row << 8) + ((row & 1) ? (in_row - 1 - i) : i)] = (uint32_t)t;
    }
}
__device__ __forceinline__ void tile_order_from_work(const uint32_t* __restrict__ work, uint32_t* __restrict__ order, int ntiles, uint32_t* s_cls /*[256]*/)
{
    tile_order_from([&](int t) { return work[t]; }, order, ntiles, s_cls);
}
// The stateless entry points (one forward + one backward per call, another camera every time: train.py) have no previous iteration
// to learn the tiles' weights from.  Their compositing BACKWARD is ordered by what the forward of the same call measured (its
// walk + ordering cost per tile, tile_work): this kernel, one workgroup in front of k_render_bwd_mfma (train step, 4 293 tiles,
// 1.5 M Gaussians: 202 against 262 us).  The weights are scaled so that the heaviest tile lands in the top class.
// One workgroup of 1 024 lanes; every tile's weight is loaded once, all loads in flight together.  Counting sort like tile_order_from, but over
// 4 096 classes: (weight scaled to 8 bits) x (tile number mod 16) -- tiles of equal weight may come in any order, and the extra bits
// keep the lanes of a wave off each other's counters (neighbouring tiles weigh about the same: with 256 classes the LDS atomics of a
// wave hit a handful of addresses and serialise -- 19 us for 4 293 tiles; three strided passes over global memory on 256 lanes: 30 us).
#define GSR_TILE_ORDER_THREADS 1024
#define GSR_TILE_ORDER_PER_LANE 16
#define GSR_STATELESS_BALANCE_MAX_TILES (GSR_TILE_ORDER_THREADS * GSR_TILE_ORDER_PER_LANE)
__device__ __forceinline__ void tile_order_block(const uint32_t* __restrict__ work, uint32_t* __restrict__ order, int ntiles)
{
    __shared__ uint32_t s_cls[4096];
    __shared__ uint16_t s_c[GSR_STATELESS_BALANCE_MAX_TILES];
    __shared__ uint32_t s_wsum[GSR_TILE_ORDER_THREADS / 64];
    __shared__ uint32_t s_max;
    const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
    if (tid == 0) s_max = 0u;
#pragma unroll
    for (int k = 0; k < 4; k++) s_cls[tid + k * GSR_TILE_ORDER_THREADS] = 0u;
    uint32_t v[GSR_TILE_ORDER_PER_LANE];
    uint32_t m = 0u;
#pragma unroll
    for (int k = 0; k < GSR_TILE_ORDER_PER_LANE; k++) {
        const int t = tid + k * GSR_TILE_ORDER_THREADS;
        v[k] = (t < ntiles) ? work[t] : 0u;
    }
#pragma unroll
    for (int k = 0; k < GSR_TILE_ORDER_PER_LANE; k++) m = max(m, v[k]);
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) m = max(m, (uint32_t)__shfl_xor((int)m, off, 64));
    __syncthreads();
    if (lane == 0) atomicMax(&s_max, m);
    __syncthreads();
    const int shift = max(0, 24 - (int)__clz(s_max | 1u));          // (work >> shift) <= 255
#pragma unroll
    for (int k = 0; k < GSR_TILE_ORDER_PER_LANE; k++) {
        const int t = tid + k * GSR_TILE_ORDER_THREADS;
        if (t < ntiles) {
            const uint32_t c = ((255u - (v[k] >> shift)) << 4) | ((uint32_t)t & 15u);      // class 0 = heaviest
            s_c[t] = (uint16_t)c;
            atomicAdd(&s_cls[c], 1u);
        }
    }
    __syncthreads();
    {   // exclusive prefix sum over the 4 096 classes: four per lane
        uint32_t c4[4], mine = 0u;
#pragma unroll
        for (int k = 0; k < 4; k++) { c4[k] = s_cls[4 * tid + k]; mine += c4[k]; }
        uint32_t incl = mine;
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
            const uint32_t o = __shfl_up(incl, off, 64);
            if (lane >= off) incl += o;
        }
        if (lane == 63) s_wsum[wv] = incl;
        __syncthreads();
        uint32_t start = incl - mine;
        for (int w = 0; w < wv; w++) start += s_wsum[w];
#pragma unroll
        for (int k = 0; k < 4; k++) { s_cls[4 * tid + k] = start; start += c4[k]; }
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < GSR_TILE_ORDER_PER_LANE; k++) {
        const int t = tid + k * GSR_TILE_ORDER_THREADS;
        if (t < ntiles) {
            const int r = (int)atomicAdd(&s_cls[s_c[t]], 1u);          // rank, heaviest first; block (r / 256) * 256 + snake(r % 256) as in tile_order_from
            const int row = r >> 8, i = r & 255;
            const int in_row = min(256, ntiles - (row << 8));
            order[(row << 8) + ((row & 1) ? (in_row - 1 - i) : i)] = (uint32_t)t;
        }
    }
}

// Launch list of the compositing kernels when heavy tiles are split (SegCtl): the tiles in the work-balanced order computed just
// before (order[]), each with nseg consecutive blocks.  A tile is split when the work its forward measured one iteration earlier
// (the longest of its four waves' walks, in groups of eight entries, plus its ordering overhead) is more than twice L = max(mean
// work, GSR_SEG_WORK_MIN): into ceil(work / L) segments -- the point is the launch's critical path, and splitting everything
// would only add pass A to everybody's bill (a scene whose tiles are all equally heavy is left alone).  The blocks must fit the
// launch (budget >= ntiles): L grows until they do.  One workgroup; the first GSR_BLOCK threads work.
#define GSR_SEG_WORK_MIN 24u
#ifndef GSR_SEG_KEYS
#define GSR_SEG_KEYS 192u          // keys per segment the launch list aims at
#endif
#ifndef GSR_SEG_SPLIT_HALVES
#define GSR_SEG_SPLIT_HALVES 2u    // a tile is split when its work exceeds this many HALVES of L = max(mean work, GSR_SEG_WORK_MIN) ...
#endif
#ifndef GSR_SEG_SPLIT_MIN_WORK
#define GSR_SEG_SPLIT_MIN_WORK 48u // ... and this much in absolute terms (groups of eight entries) ...
#endif
#ifndef GSR_SEG_SPLIT_SURE
#define GSR_SEG_SPLIT_SURE 3u      // ... or, whatever its absolute size, this many halves of L
#endif
// (round 5, tools/dbg/timeline.py on S-room-640: with the threshold at 2 L the launches ended with a dozen UNSPLIT tiles of 1-2 L that had
// been running since the first microsecond -- a workgroup shares its SIMDs with four others, so a tile of 800 entries in one 8x8 block
// is a 190 us chain while the sum of all lifetimes is worth 110 us of the machine.  Thresholds measured (it/s: S-room-640 / S-1M-640-object
// / S-1M-640): 2 L 1 545 / 3 938 / 6 700; 1.5 L 1 601 / 4 072 / 6 759; 1 L 1 772 / 4 062 / 6 503 (eight tiles of the uniform cloud split
// in two: a split tile is a longer chain than the same tile whole unless it is heavy in absolute terms); 1 L above 48 groups, 1.5 L
// below, room for 3 blocks per tile: 1 847 / 4 077 / 6 734 -- kept.  Raising the wave priority of the launch's front (s_setprio) did nothing.)
#ifndef GSR_BWD_SEG_MERGE
#define GSR_BWD_SEG_MERGE 1u       // forward segments per workgroup of the backward compositing kernel (measured, S-1M-640-object: 1 -> 93 us, 2 -> 106, 3 -> 129)
#endif
#define GSR_SEG_MAX 32             // segments per tile at most
#define GSR_SEG_BUILD_MAX_TILES 4096      // (16 launch positions per thread, kept in registers)
__device__ __forceinline__ void seg_list_build(const uint32_t* __restrict__ work, const uint32_t* __restrict__ order, uint32_t* __restrict__ list,
                                               uint32_t* __restrict__ nosplit, int ntiles, int budget, const uint32_t* __restrict__ len,
                                               uint32_t* __restrict__ host_total, bool split_ok)
{
    __shared__ uint32_t s_sum[4];
    const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
    const bool act = tid < GSR_BLOCK;
    auto block_sum = [&](uint32_t v) -> uint32_t {          // every thread of the workgroup must call
#pragma unroll
        for (int off = 32; off > 0; off >>= 1) v += (uint32_t)__shfl_xor((int)v, off, 64);
        __syncthreads();
        if (act && lane == 0) s_sum[wv] = v;
        __syncthreads();
        return s_sum[0] + s_sum[1] + s_sum[2] + s_sum[3];
    };
    // launch positions are dealt to the threads in contiguous chunks (a prefix sum over the chunks gives every tile its first block);
    // a thread's tiles, their work and hold counters are read once, all loads in flight together
    constexpr int kPer = GSR_SEG_BUILD_MAX_TILES / GSR_BLOCK;
    const int chunk = (ntiles + GSR_BLOCK - 1) / GSR_BLOCK;
    const int p0 = min(tid * chunk, ntiles), np = act ? min(chunk, ntiles - p0) : 0;
    uint32_t tl[kPer], wk[kPer], hold[kPer], ln[kPer];
#pragma unroll
    for (int i = 0; i < kPer; i++) tl[i] = (i < np) ? order[p0 + i] : 0u;
#pragma unroll
    for (int i = 0; i < kPer; i++) { wk[i] = (i < np) ? work[tl[i]] : 0u; hold[i] = (i < np) ? nosplit[tl[i]] : 0u; ln[i] = (i < np) ? len[tl[i]] : 0u; }
    uint32_t mine = 0u;
#pragma unroll
    for (int i = 0; i < kPer; i++) mine += wk[i];
    const uint32_t all_work = block_sum(mine);
    const uint32_t mean = all_work / (uint32_t)max(ntiles, 1);
    uint32_t L = split_ok ? max(mean, GSR_SEG_WORK_MIN) : 0x3FFFFFFFu;      // (!split_ok: the list is the plain order, one block per tile)
    // A SKEWED launch -- a tenth or more of all work sits in tiles above 2 L -- ends with a long tail of its upper-middle tiles as well
    // (see GSR_SEG_SPLIT_HALVES): there the threshold drops to 1 L / 1.5 L.  A launch of roughly equal tiles has half of them above the mean
    // by definition; splitting those buys nothing (S-1M-640-walls in the iterations right after a complete-list forward: 570 of 1 200 tiles).
    uint32_t heavy = 0u;
#pragma unroll
    for (int i = 0; i < kPer; i++) heavy += (wk[i] > 2u * L) ? wk[i] : 0u;
    heavy = block_sum(heavy);
    const bool skewed = (unsigned long long)heavy * 10ull >= (unsigned long long)all_work;
    const uint32_t halves = skewed ? GSR_SEG_SPLIT_HALVES : 4u, sure = skewed ? GSR_SEG_SPLIT_SURE : 4u;
    // (WHETHER a tile is split is a matter of its work against the mean; into HOW MANY segments also of its list's length: a segment of
    // up to GSR_BLOCK keys sorts in registers and is staged once for both passes -- measured, S-1M-640-object / S-room-640: segments of
    // 500 - 1 300 keys cost more than a whole median tile, most of it barriers between their staging batches and the LDS sort)
    uint32_t Lk = GSR_SEG_KEYS;
    auto nseg_of = [&](uint32_t w, uint32_t h, uint32_t n) -> uint32_t {
        if (2u * w <= halves * L || (w <= GSR_SEG_SPLIT_MIN_WORK && 2u * w <= sure * L) || h != 0u) return 1u;
        return min((uint32_t)GSR_SEG_MAX, max((w + L - 1u) / L, (n + Lk - 1u) / Lk));
    };
    uint32_t total = 0u, local = 0u;
    for (int round = 0; round < 16; round++) {
        local = 0u;
#pragma unroll
        for (int i = 0; i < kPer; i++) local += (i < np) ? nseg_of(wk[i], hold[i], ln[i]) : 0u;
        total = block_sum(local);
        if (total <= (uint32_t)budget) break;
        L += (L >> 1) + 1u;          // (the blocks must fit the launch: fewer, longer segments)
        Lk += (Lk >> 1);
    }
    if (total > (uint32_t)budget) {          // (cannot happen with budget >= ntiles; then nobody is split)
        L = 0x3FFFFFFFu;
        local = (uint32_t)np;
        total = block_sum(local);
    }
    uint32_t incl = local;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const uint32_t o = (uint32_t)__shfl_up((int)incl, off, 64);
        if (lane >= off) incl += o;
    }
    __syncthreads();
    if (act && lane == 63) s_sum[wv] = incl;
    __syncthreads();
    uint32_t at = incl - local;
    for (int w = 0; act && w < wv; w++) at += s_sum[w];
#pragma unroll
    for (int i = 0; i < kPer; i++)
        if (i < np) {
            const uint32_t k = nseg_of(wk[i], hold[i], ln[i]);
            for (uint32_t q = 0; q < k; q++) list[at + q] = tl[i] | (q << 16) | (k << 24);
            at += k;
            if (hold[i] != 0u) nosplit[tl[i]] = hold[i] - 1u;
        }
    for (int b = (int)total + tid; b < budget; b += blockDim.x) list[b] = 0xFFFFFFFFu;
    if (host_total != nullptr && tid == 0) *reinterpret_cast<volatile uint32_t*>(host_total) = total;
}

// What the walk keeps per Gaussian between its passes over the image (registers): the span test without the terms only
// needed once, the clipped rectangle, the key.
struct WalkItem {
    float mx, my, at, B, det, dye, invA;           // at = A * twoq
    int x0, y0, x1, y1;                            // clipped tile rectangle; x1 == x0: nothing to do
    unsigned long long key;
    bool all;                                      // conic not positive definite: every tile of the rectangle
};
__device__ __forceinline__ void item_span(const WalkItem& t, int ty, int& lo, int& hi)      // row_span on the cached terms
{
    if (t.all) { lo = t.x0; hi = t.x1 - 1; return; }
    lo = 1; hi = 0;
    const float dyh = t.my - (float)(ty * GSR_TILE), dyl = dyh - (float)(GSR_TILE - 1);
    const float dy1 = fminf(dyh, fmaxf(dyl, t.dye)), dy2 = fminf(dyh, fmaxf(dyl, -t.dye));
    const float disc1 = t.at - t.det * dy1 * dy1, disc2 = t.at - t.det * dy2 * dy2;
    if (fminf(disc1, disc2) < -1e-3f * t.at) return;
    const float dmax = (__builtin_amdgcn_sqrtf(fmaxf(disc1, 0.f)) - t.B * dy1) * t.invA;
    const float dmin = (-__builtin_amdgcn_sqrtf(fmaxf(disc2, 0.f)) - t.B * dy2) * t.invA;
    const float pa = t.mx - dmax - 0.01f, pb = t.mx - dmin + 0.01f;
    lo = max(t.x0, (int)ceilf((pa - (float)(GSR_TILE - 1)) * (1.f / GSR_TILE)));
    hi = min(t.x1 - 1, (int)floorf(pb * (1.f / GSR_TILE)));
}
// Upper bound on sqrt(lambda_max(Sigma)) of a symmetric positive semi-definite 3x3 matrix given by its six unique entries -- the
// "largest scale" of a Gaussian whatever produced its covariance (a quaternion that is not normalised is used as given,
// forward.cu:127: its R is not orthogonal and max(scale) says nothing about Sigma).  lambda_max <= min(Frobenius norm,
// largest absolute row sum); exact for a diagonal Sigma, within 3^(1/4) of the truth in the worst case.  NaN / Inf propagate
// (the caller then leaves the decision to the exact code).
__device__ __forceinline__ float sigma_extent_bound(const float* c6)
{
    const float f2 = c6[0] * c6[0] + c6[3] * c6[3] + c6[5] * c6[5] + 2.f * (c6[1] * c6[1] + c6[2] * c6[2] + c6[4] * c6[4]);
    const float r0 = fabsf(c6[0]) + fabsf(c6[1]) + fabsf(c6[2]), r1 = fabsf(c6[1]) + fabsf(c6[3]) + fabsf(c6[4]),
                r2 = fabsf(c6[2]) + fabsf(c6[4]) + fabsf(c6[5]);
    const float lmax = fminf(sqrtf(f2), fmaxf(r0, fmaxf(r1, r2)));
    return sqrtf(lmax) * 1.00001f;
}
// Upper bound on |W|_2^2 of the view matrix's 3x3 block (1 for a rigid camera pose, up to rounding; the bound must hold for
// whatever the caller passes): largest absolute row sum of W W^T.
__device__ __forceinline__ float view_norm2_bound(const float* view)
{
    const float r0[3] = {view[0], view[4], view[8]}, r1[3] = {view[1], view[5], view[9]}, r2[3] = {view[2], view[6], view[10]};
    const float g00 = r0[0] * r0[0] + r0[1] * r0[1] + r0[2] * r0[2], g11 = r1[0] * r1[0] + r1[1] * r1[1] + r1[2] * r1[2],
                g22 = r2[0] * r2[0] + r2[1] * r2[1] + r2[2] * r2[2];
    const float g01 = fabsf(r0[0] * r1[0] + r0[1] * r1[1] + r0[2] * r1[2]), g02 = fabsf(r0[0] * r2[0] + r0[1] * r2[1] + r0[2] * r2[2]),
                g12 = fabsf(r1[0] * r2[0] + r1[1] * r2[1] + r1[2] * r2[2]);
    return fmaxf(g00 + g01 + g02, fmaxf(g01 + g11 + g12, g02 + g12 + g22)) * 1.0001f;
}
// The conservative test of k_preprocess_lean for one Gaussian in front of the near plane (pview.z > 0.2): can it still be
// binned into a tile under the current depth bounds?  false = settled (behind the bound of every superblock a rectangle
// CONTAINING its exact tile rectangle overlaps, or that rectangle is empty).
//   cov2D = J W Sigma W^T J^T  =>  lambda_max(cov2D + 0.3 I) <= |J|_F^2 |W|_2^2 lambda_max(Sigma) + 0.3, J the 2x3 perspective
//   Jacobian with the clamped x/z, y/z of forward.cu:90-96; the reference's radius uses mid + sqrt(max(0.1, mid^2 - det)) <=
//   lambda_max + sqrt(0.1); together <= jn2 wn2 seff^2 + 0.62 (0.95 here).  seff = sigma_extent_bound of the Gaussian's actual
//   Sigma, wn2 = view_norm2_bound: no assumption on the quaternion, the scale modifier or the pose matrix.  Hardware
//   reciprocals and fp32 pixel centres are covered by a 0.2 % + 0.2 % + two-pixel allowance; a bound of a million pixels or
//   more (or NaN) is not trusted at all: candidate, the exact code decides.
// zbc: the superblock bounds; MIP: followed (k_preprocess_lean's copy in LDS, build_bound_pyramid) by coarser levels, each the
// maximum over 2 x 2 cells of the one below, down to a level of at most 3 x 3 cells.  The bound of a rectangle is then the maximum
// over at most 3 x 3 cells of the finest level on which it spans no more than that -- nine independent LDS reads.  (Round 2
// walked the rectangle's superblocks one by one: a loop of up to 80 dependent LDS reads whose trip count is the LARGEST of the
// wave's 64 lanes -- one big splat near the camera among a wave's 256 Gaussians, which half of the waves have, and the
// conservative pass took 45 k cycles instead of 22 k: that pass, not the exact one, was the kernel's slow tail,
// profiles/r03_phase_clocks.md.)  Coarser cells only make the test more conservative.
// (largest superblock bound under the non-empty tile rectangle [x0, x1) x [y0, y1))
// (shift: 2 = the finest level's cells are 4 x 4-tile superblocks, 0 = they are tiles -- round 5: a splat inside a dense object one
// superblock wide saw its neighbours' deep background bounds and stayed a candidate: half a million candidates per iteration on
// S-1M-640-object, the preprocess kernel at 72 us against 35 on the uniform cloud)
template <bool MIP>
__device__ __forceinline__ float rect_bound_max(const float* zbc, int sbx, int sby, int x0, int y0, int x1, int y1, int shift = 2)
{
    float zc = 0.f;
    if (MIP) {
        int sx0 = x0 >> shift, sx1 = (x1 - 1) >> shift, sy0 = y0 >> shift, sy1 = (y1 - 1) >> shift, w = sbx, h = sby, off = 0;
        while (sx1 - sx0 > 2 || sy1 - sy0 > 2) {
            off += w * h; w = (w + 1) >> 1; h = (h + 1) >> 1;
            sx0 >>= 1; sx1 >>= 1; sy0 >>= 1; sy1 >>= 1;
        }
#pragma unroll
        for (int dy = 0; dy < 3; dy++)
#pragma unroll
            for (int dx = 0; dx < 3; dx++) zc = fmaxf(zc, zbc[off + min(sy0 + dy, sy1) * w + min(sx0 + dx, sx1)]);
    } else {
        for (int sy = y0 >> shift; sy <= (y1 - 1) >> shift; sy++)
            for (int sx = x0 >> shift; sx <= (x1 - 1) >> shift; sx++) zc = fmaxf(zc, zbc[sy * sbx + sx]);
    }
    return zc;
}
template <bool MIP>
__device__ __forceinline__ bool lean_candidate(const PreArgs& a, float3 p, float3 pview, float seff, float wn2, const float* zbc)
{
    const float4 ph = xform4x4(p, a.proj);
    const float pw = __builtin_amdgcn_rcpf(ph.w + 0.0000001f);
    const float rz = __builtin_amdgcn_rcpf(pview.z);
    const float ccx = fminf(1.3f * a.tanx, fmaxf(-1.3f * a.tanx, pview.x * rz));
    const float ccy = fminf(1.3f * a.tany, fmaxf(-1.3f * a.tany, pview.y * rz));
    const float jx = a.fx * rz, jy = a.fy * rz;
    const float jn2 = (jx * jx * (1.f + ccx * ccx) + jy * jy * (1.f + ccy * ccy)) * wn2;
    const float rb = ceilf(3.f * __builtin_amdgcn_sqrtf((jn2 * seff) * seff * 1.002f + 0.95f) * 1.002f) + 2.f;
    if (!(rb < 1.0e6f)) return true;
    const float pxf = ((ph.x * pw + 1.f) * (float)a.W - 1.f) * 0.5f, pyf = ((ph.y * pw + 1.f) * (float)a.H - 1.f) * 0.5f;
    int x0, y0, x1, y1;
    get_rect(pxf, pyf, (int)rb, a.gx, a.gy, x0, y0, x1, y1);
    if ((x1 - x0) * (y1 - y0) == 0) return false;
    const float zc = a.pyr_tiles ? rect_bound_max<MIP>(zbc, a.gx, a.gy, x0, y0, x1, y1, 0) : rect_bound_max<MIP>(zbc, a.sbx, a.sby, x0, y0, x1, y1, 2);
    return !(pview.z > zc * a.zb_mul + a.zb_add);
}
// Appends the coarser levels behind the sbx x sby superblock bounds in s (LDS, all threads of the workgroup; s[0, sbx * sby) staged
// and a barrier passed): level l + 1 = maxima over 2 x 2 cells of level l, until a level has at most 3 x 3 cells.
__device__ __forceinline__ void build_bound_pyramid(float* s, int sbx, int sby)
{
    int w = sbx, h = sby, off = 0;
    while (w > 3 || h > 3) {
        const int nw = (w + 1) >> 1, nh = (h + 1) >> 1, noff = off + w * h;
        for (int i = threadIdx.x; i < nw * nh; i += blockDim.x) {
            const int cx = i % nw, cy = i / nw, x0 = 2 * cx, y0 = 2 * cy, x1 = min(x0 + 1, w - 1), y1 = min(y0 + 1, h - 1);
            s[noff + i] = fmaxf(fmaxf(s[off + y0 * w + x0], s[off + y0 * w + x1]), fmaxf(s[off + y1 * w + x0], s[off + y1 * w + x1]));
        }
        __syncthreads();
        off = noff; w = nw; h = nh;
    }
}
static inline size_t bound_pyramid_floats(int sbx, int sby)
{
    size_t n = (size_t)sbx * sby;
    int w = sbx, h = sby;
    while (w > 3 || h > 3) { w = (w + 1) >> 1; h = (h + 1) >> 1; n += (size_t)w * h; }
    return n;
}

// Everything k_preprocess does for ONE Gaussian (lane) once its index is known: exact geometry, the bound tests, binning on
// the by-tile path, survivor list, stale gradient rows.  Called with idx = the thread's global index (k_preprocess) or a
// compacted candidate (k_preprocess_lean); wave-level pieces (cooperative walks, list appends) work on any 64 lanes.
// FLAT (k_preprocess_lean: every live lane of the wave has a footprint to walk): the tile instances of all lanes are laid end to
// end (prefix sum of the clipped rectangles' areas) and taken 64 at a time -- each lane finds whose instance it got (binary
// search in the wave's prefix array), fetches that Gaussian's terms from the owning lane (ds_bpermute) and tests / appends
// ONE tile, so that a round is one set of independent bound loads and returning atomics instead of a chain of them per
// Gaussian.  s_flat: 128 words of LDS per wave (prefix array, per-owner counts).
// wout (nullable; complete lists binned by the same kernel, k_preprocess_bin): receives what the row walk needs -- span terms, the
// clipped rectangle, the key -- straight from this lane's registers (x1 == x0: nothing to walk).
template <bool FLAT>
__device__ __forceinline__ void preprocess_one(const PreArgs& a, const int idx, const bool live, const float* s_zbc, const int tid, const uint32_t sublist,
                                               uint32_t* s_flat = nullptr, WalkItem* wout = nullptr)
{
#if GSR_TIMING
    const long long tp0_ = clock64();
#endif
    bool vis = false, coop = false, own = false, store_cov = false;
    float3 p = make_float3(0.f, 0.f, 0.f);
    TileTest tt = {};
    int rx0 = 0, ry0 = 0, rx1 = 0, ry1 = 0;
    float zv = 0.f;
    uint32_t cnt = 0;

    // FLAT (the compacted candidates of k_preprocess_lean: every live lane is in front of the camera and will need all of it):
    // everything the lane reads about its Gaussian is requested up front -- one round trip instead of a chain of four (mean ->
    // covariance -> opacity -> SH row; the wave's lifetime is these dependent round trips, not arithmetic).  The SH row is only
    // touched (its two cache lines), not held in registers.
    float cov_h[6] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f}, opac_h = 0.f, sh_touch0 = 0.f, sh_touch1 = 0.f;
    const bool hoist = FLAT && live && a.cov3D_pre != nullptr && !a.cov_all;
    if (hoist) {
#pragma unroll
        for (int i = 0; i < 6; i++) cov_h[i] = a.cov3D_pre[6 * (size_t)idx + i];
        opac_h = a.opac[idx];
        if (a.sh_here && a.shs != nullptr && a.M >= 16) { sh_touch0 = a.shs[(size_t)idx * a.M * 3]; sh_touch1 = a.shs[(size_t)idx * a.M * 3 + 32]; }
    }
    if (live) {
        a.radii[idx] = 0;
        a.tiles_touched[idx] = 0;
        if (a.n_touched != nullptr) a.n_touched[idx] = 0;
        p = make_float3(a.means[3 * idx], a.means[3 * idx + 1], a.means[3 * idx + 2]);
        const float4 ph = xform4x4(p, a.proj);
        const float pw = 1.0f / (ph.w + 0.0000001f);
        const float3 pproj = make_float3(ph.x * pw, ph.y * pw, ph.z * pw);
        const float3 pview = xform4x3(p, a.view);
        float cov6[6];
        if (a.cov_all) {
            // native loop, first forward of a refinement: the map does not change while the pose is refined, so the
            // 3D covariances are computed for EVERY Gaussian now (also the ones culled at this pose) and the later
            // iterations read them back (cov3D_pre = this buffer) instead of rebuilding them from scale and rotation
            float s3[3] = {a.scales[3 * idx], a.scales[3 * idx + 1], a.scales[3 * idx + 2]};
            const float4 q = reinterpret_cast<const float4*>(a.rots)[idx];
            float q4[4] = {q.x, q.y, q.z, q.w};
            cov3d_from_scale_rot(s3, a.mod, q4, cov6);
#pragma unroll
            for (int i = 0; i < 6; i++) a.cov3D[6 * (size_t)idx + i] = cov6[i];
            if (a.lam != nullptr) reinterpret_cast<float4*>(a.lam)[idx] = make_float4(p.x, p.y, p.z, sigma_extent_bound(cov6));
        }
        if (pview.z > 0.2f) {     // near cull (auxiliary.h:150)
            if (a.cov_all) {
            } else if (hoist) {
#pragma unroll
                for (int i = 0; i < 6; i++) cov6[i] = cov_h[i];
            } else if (a.cov3D_pre != nullptr) {
#pragma unroll
                for (int i = 0; i < 6; i++) cov6[i] = a.cov3D_pre[6 * (size_t)idx + i];
            } else {
                float s3[3] = {a.scales[3 * idx], a.scales[3 * idx + 1], a.scales[3 * idx + 2]};
                const float4 q = reinterpret_cast<const float4*>(a.rots)[idx];
                float q4[4] = {q.x, q.y, q.z, q.w};
                cov3d_from_scale_rot(s3, a.mod, q4, cov6);
                store_cov = true;          // (kept for the backward pass -- of the Gaussians that turn out to be visible only)
            }
            Cov2DTerms ct;
            cov2d_terms(p, a.fx, a.fy, a.tanx, a.tany, cov6, a.view, ct);
            const float cx = ct.cov.m[0][0] + 0.3f, cy = ct.cov.m[0][1], cz = ct.cov.m[1][1] + 0.3f;
            const float det = (cx * cz - cy * cy);
            if (det != 0.0f) {
                const float det_inv = 1.f / det;
                const float3 conic = make_float3(cz * det_inv, -cy * det_inv, cx * det_inv);
                const float mid = 0.5f * (cx + cz);
                const float lambda1 = mid + sqrtf(fmaxf(0.1f, mid * mid - det));
                const float lambda2 = mid - sqrtf(fmaxf(0.1f, mid * mid - det));
                const float my_radius = ceilf(3.f * sqrtf(fmaxf(lambda1, lambda2)));
                const float2 pix = make_float2(ndc2pix(pproj.x, a.W), ndc2pix(pproj.y, a.H));
                int x0, y0, x1, y1;
                get_rect(pix.x, pix.y, (int)my_radius, a.gx, a.gy, x0, y0, x1, y1);
                if ((x1 - x0) * (y1 - y0) != 0) {
                    vis = true;
                    const float opacity = hoist ? opac_h : a.opac[idx];
                    a.radii[idx] = (int)my_radius;
                    if (store_cov) {
#pragma unroll
                        for (int i = 0; i < 6; i++) a.cov3D[6 * (size_t)idx + i] = cov6[i];
                    }
                    {
                        float4* rec = reinterpret_cast<float4*>(a.rec + (size_t)idx * GSR_REC_STRIDE);
                        rec[0] = make_float4(pix.x, pix.y, (-GSR_LOG2E) * conic.y, (-0.5f * GSR_LOG2E) * conic.z);
                        rec[1] = make_float4((-0.5f * GSR_LOG2E) * conic.x, opacity, pview.z, 0.f);
                        if (a.colors_pre != nullptr) rec[2] = make_float4(a.colors_pre[3 * idx], a.colors_pre[3 * idx + 1], a.colors_pre[3 * idx + 2], 1.f);
                        else if (a.lazy_sh) rec[2] = make_float4(0.f, 0.f, 0.f, 0.f);      // (.w = 0: colour not evaluated yet, see LazySH)
                    }
                    a.rects[idx] = make_ushort4((unsigned short)x0, (unsigned short)y0, (unsigned short)x1, (unsigned short)y1);
                    // exact count of tiles this splat can change
                    tt = make_tile_test(pix, conic, opacity);
                    rx0 = x0; ry0 = y0; rx1 = x1; ry1 = y1; zv = pview.z;
                    clip_rect(tt, rx0, ry0, rx1, ry1);      // (walked below; the stored rectangle stays the reference's)
                    bool far_everywhere = false;
                    if (a.zb != nullptr) {
                        // behind the bound of every superblock the rectangle overlaps => behind every tile's bound
                        // (s_zbc: the bounds in LDS with the coarser levels behind them, build_bound_pyramid; otherwise global memory)
                        const float zc = (s_zbc != nullptr && a.zbc_lds > 0) ? (a.pyr_tiles ? rect_bound_max<true>(s_zbc, a.gx, a.gy, x0, y0, x1, y1, 0)
                                                                                             : rect_bound_max<true>(s_zbc, a.sbx, a.sby, x0, y0, x1, y1, 2))
                                                                              : rect_bound_max<false>(a.zbc, a.sbx, a.sby, x0, y0, x1, y1, 2);
                        far_everywhere = pview.z > zc * a.zb_mul + a.zb_add;
                    }
                    if (a.bins == nullptr || wout != nullptr) {
                        // complete lists: k_tile_count / k_tile_emit (or the second half of k_preprocess_bin) walk the tiles; here
                        // only "can this splat reach any pixel"
                        cnt = tt.none ? 0u : 1u;
                        if (wout != nullptr && cnt != 0u) {
                            wout->x0 = rx0; wout->y0 = ry0; wout->x1 = rx1; wout->y1 = ry1;
                            wout->mx = tt.mx; wout->my = tt.my; wout->at = tt.A * tt.twoq; wout->B = tt.B; wout->det = tt.det; wout->dye = tt.dye;
                            wout->invA = tt.invA; wout->all = !tt.cull;
                            wout->key = ((unsigned long long)__float_as_uint(pview.z) << 32) | (uint32_t)idx;
                        }
                    } else if (!far_everywhere) {
                        if ((rx1 - rx0) * (ry1 - ry0) > GSR_COOP_AREA) coop = true;      // whole wave helps below
                        else own = true;
                    }
                }
            }
        }
    }
#if GSR_TIMING
    const long long tp1_ = clock64();
#endif
    if (FLAT) {
        const int lane = tid & 63;
        const bool walker = own || coop;
        const int area = walker ? (rx1 - rx0) * (ry1 - ry0) : 0;
        int incl = area;
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
            const int o = __shfl_up(incl, off, 64);
            if (lane >= off) incl += o;
        }
        const int total = __builtin_amdgcn_readlane(incl, 63);
        uint32_t* pref = s_flat;            // first instance slot of lane's Gaussian (lanes without a footprint share their successor's)
        uint32_t* ocnt = s_flat + 64;       // instances appended per owner
        pref[lane] = (uint32_t)(incl - area);
        ocnt[lane] = 0u;
        __builtin_amdgcn_wave_barrier();
#define GSR_PERM_F(v, src) __uint_as_float((uint32_t)__builtin_amdgcn_ds_bpermute((src) << 2, (int)__float_as_uint(v)))
#define GSR_PERM_I(v, src) __builtin_amdgcn_ds_bpermute((src) << 2, (int)(v))
        // four steps (256 instances) per round, phase by phase: every bound load of the round is in flight before the first
        // is needed, likewise the returning atomics on the tile cursors
#if GSR_TIMING
        if ((tid & 63) == 0 && s_flat != nullptr) s_flat[128] += (uint32_t)total;      // (diagnostics: instances walked by this wave)
#endif
        for (int u0 = 0; u0 < total; u0 += 4 * 64) {
            int f_tile[4], f_src[4]; float f_z[4], f_zb[4]; uint32_t f_id[4]; bool f_in[4];
#pragma unroll
            for (int k = 0; k < 4; k++) {
                f_in[k] = false; f_tile[k] = 0; f_zb[k] = 0.f; f_z[k] = 0.f; f_id[k] = 0u; f_src[k] = 0;
                if (u0 + 64 * k >= total) continue;          // (wave-uniform)
                const int u = u0 + 64 * k + lane;
                const bool act = u < total;
                int src = 0;
                if (act) {
#pragma unroll
                    for (int step = 32; step > 0; step >>= 1)
                        if (pref[src + step] <= (uint32_t)u) src += step;
                }
                TileTest bt;
                bt.mx = GSR_PERM_F(tt.mx, src); bt.my = GSR_PERM_F(tt.my, src); bt.A = GSR_PERM_F(tt.A, src); bt.B = GSR_PERM_F(tt.B, src);
                bt.det = GSR_PERM_F(tt.det, src); bt.twoq = GSR_PERM_F(tt.twoq, src); bt.dye = GSR_PERM_F(tt.dye, src); bt.invA = GSR_PERM_F(tt.invA, src);
                bt.C = 0.f; bt.dxe = 0.f; bt.dyext = 0.f;      // (not used by row_span)
                const int flags = GSR_PERM_I((int)tt.cull | ((int)tt.none << 1), src);
                bt.cull = (flags & 1) != 0; bt.none = (flags & 2) != 0;
                f_z[k] = GSR_PERM_F(zv, src);
                const int bx0 = GSR_PERM_I(rx0, src), by0 = GSR_PERM_I(ry0, src), bx1 = GSR_PERM_I(rx1, src);
                f_id[k] = (uint32_t)GSR_PERM_I(idx, src);
                f_src[k] = src;
                if (act) {
                    const int bw = bx1 - bx0, t = u - (int)pref[src];
                    const int row = (int)((float)t * __builtin_amdgcn_rcpf((float)bw) + 0.001f);      // t / bw (corrected below)
                    int ry = row, rxo = t - row * bw;
                    if (rxo < 0) { ry--; rxo += bw; } else if (rxo >= bw) { ry++; rxo -= bw; }
                    const int y = by0 + ry, x = bx0 + rxo;
                    int lo, hi;
                    row_span(bt, y, bx0, bx1, lo, hi);
                    f_tile[k] = y * a.gx + x;
                    f_in[k] = x >= lo && x <= hi;
                    if (f_in[k]) f_zb[k] = a.zb[f_tile[k]];
                }
            }
            uint32_t f_pos[4];
#pragma unroll
            for (int k = 0; k < 4; k++) {
                // behind everything this tile needed last iteration (+ margin): speculatively dropped
                f_in[k] = f_in[k] && f_z[k] <= f_zb[k] * a.zb_mul + a.zb_add;
                f_pos[k] = (uint32_t)a.bin_cap;
#if GSR_TIMING
                {   // (diagnostics: appends of this wave, and how many of them went to tiles without a depth bound)
                    const uint32_t n_app = (uint32_t)__popcll(__ballot(f_in[k])), n_inf = (uint32_t)__popcll(__ballot(f_in[k] && !(f_zb[k] < __builtin_huge_valf())));
                    if ((tid & 63) == 0 && s_flat != nullptr) { s_flat[133] += n_app; s_flat[134] += n_inf; }
                }
#endif
                if (f_in[k]) {
                    atomicAdd(&ocnt[f_src[k]], 1u);
                    // (appends of one wave to the SAME tile grouped into one atomic -- a wave-uniform loop of ballots over up to 12 / 32 distinct
                    // tiles per sub-round -- were measured in round 5 for S-1M-640-object, whose hot tiles take ~4 000 appends per iteration:
                    // this kernel 75 -> 78 / 86 us there, 36 -> 44 / 47 us on the uniform cloud.  Round 6 looked at the launches behind a failed
                    // forward on that scene (2.1 ms and 0.73 ms instead of 30 us: a silhouette tile without a bound takes the 100-190 k splats
                    // of the object behind it, one cursor, ~11 ns per same-address atomic -- tools/micro/atomic_scope.hip, tools/dbg/kt_longest.py,
                    // lean_cold.py).  Three remedies built and measured, none kept: a coherent read of the cursor in front of the atomic
                    // (skip once the bin has overflowed: the reads queue at the same memory-side word), one atomic per (wave, unbounded
                    // tile) (a wave holds ~46 of those appends spread over its sub-rounds: a serial loop over the distinct tiles costs more
                    // than it merges -- S-room-640 174 -> 198 us), and one dominant-tile group per sub-round (fewer than sixteen lanes share
                    // a tile there: never taken).  The list of such a tile does not fit its bin anyway -- the call ends on the exact path.)
                    f_pos[k] = atomicAdd(&a.tile_cursor[f_tile[k] * GSR_CURSOR_STRIDE], 1u);
                }
            }
#pragma unroll
            for (int k = 0; k < 4; k++)
                if (f_pos[k] < (uint32_t)a.bin_cap)
                    a.bins[(size_t)f_tile[k] * (a.bin_cap + GSR_BIN_PAD) + f_pos[k]] = ((unsigned long long)__float_as_uint(f_z[k]) << 32) | f_id[k];
        }
#undef GSR_PERM_F
#undef GSR_PERM_I
        __builtin_amdgcn_wave_barrier();
        if (walker) cnt = ocnt[lane];
    }
    if (!FLAT && own) {      // small footprint: the lane walks its own rectangle
        for (int y = ry0; y < ry1; y++) {
            int lo, hi;
            row_span(tt, y, rx0, rx1, lo, hi);
            // behind everything this tile needed last iteration (+ margin): speculatively dropped
            for (int x = lo; x <= hi; x++)
                if (zv <= a.zb[y * a.gx + x] * a.zb_mul + a.zb_add) {
                    cnt++;
                    const int tile = y * a.gx + x;
                    const uint32_t pos = atomicAdd(&a.tile_cursor[tile * GSR_CURSOR_STRIDE], 1u);
                    if (pos < (uint32_t)a.bin_cap)
                        a.bins[(size_t)tile * (a.bin_cap + GSR_BIN_PAD) + pos] = ((unsigned long long)__float_as_uint(zv) << 32) | (uint32_t)idx;
                }
        }
    }
    if (!FLAT && a.bins != nullptr) {
        // Large footprints: the 64 lanes of the wave walk the rectangle together (one tile per lane), so no lane
        // is left issuing hundreds of dependent atomics on its own.
        const int lane = tid & 63;
        unsigned long long todo = __ballot(coop);
        while (todo != 0ull) {
            const int src = (int)__builtin_ctzll(todo);
            todo &= todo - 1ull;
            TileTest bt;
#define GSR_BCAST_F(v) __uint_as_float(__builtin_amdgcn_readlane((int)__float_as_uint(v), src))
            bt.mx = GSR_BCAST_F(tt.mx); bt.my = GSR_BCAST_F(tt.my); bt.A = GSR_BCAST_F(tt.A); bt.B = GSR_BCAST_F(tt.B);
            bt.C = GSR_BCAST_F(tt.C); bt.det = GSR_BCAST_F(tt.det); bt.twoq = GSR_BCAST_F(tt.twoq);
            bt.dxe = GSR_BCAST_F(tt.dxe); bt.dye = GSR_BCAST_F(tt.dye); bt.invA = GSR_BCAST_F(tt.invA);
            bt.cull = __builtin_amdgcn_readlane((int)tt.cull, src) != 0;
            bt.none = __builtin_amdgcn_readlane((int)tt.none, src) != 0;
            const float bz = GSR_BCAST_F(zv);
#undef GSR_BCAST_F
            const int bx0 = __builtin_amdgcn_readlane(rx0, src), by0 = __builtin_amdgcn_readlane(ry0, src);
            const int bx1 = __builtin_amdgcn_readlane(rx1, src), by1 = __builtin_amdgcn_readlane(ry1, src);
            const uint32_t bidx = (uint32_t)__builtin_amdgcn_readlane(idx, src);
            const int bw = bx1 - bx0, area = bw * (by1 - by0);
            uint32_t c_cnt = 0;
            for (int t0 = 0; t0 < area; t0 += 64) {
                const int t = t0 + lane;
                bool in_span = false, pass = false;
                if (t < area) {
                    const int y = by0 + t / bw, x = bx0 + (t - (t / bw) * bw);
                    int lo, hi;
                    row_span(bt, y, bx0, bx1, lo, hi);
                    in_span = x >= lo && x <= hi;
                    pass = in_span && bz <= a.zb[y * a.gx + x] * a.zb_mul + a.zb_add;
                    if (pass) {
                        const int tile = y * a.gx + x;
                        const uint32_t pos = atomicAdd(&a.tile_cursor[tile * GSR_CURSOR_STRIDE], 1u);
                        if (pos < (uint32_t)a.bin_cap)
                            a.bins[(size_t)tile * (a.bin_cap + GSR_BIN_PAD) + pos] = ((unsigned long long)__float_as_uint(bz) << 32) | bidx;
                    }
                }
                c_cnt += (uint32_t)__popcll(__ballot(pass));
            }
            if (lane == src) cnt = c_cnt;
        }
    }
#if GSR_TIMING
    const long long tp2_ = clock64();
#endif
    if (vis) {
        // (what was dropped is not recorded: an instance can only be dropped from a tile whose bound is finite, and the
        // compositing kernel treats every such tile that ends unsaturated as a failed speculation)
        a.tiles_touched[idx] = cnt;
    }
    // survivors -> this workgroup's work list (see SurvLists)
    const bool surv = vis && cnt != 0u;
    if (a.surv.ids != nullptr) {
        const unsigned long long mk = __ballot(surv);
        if (mk != 0ull) {
            const int lane = tid & 63;
            const uint32_t sl = sublist;
            uint32_t at = 0u;
            if (lane == 0) at = atomicAdd(&a.surv.n[sl * GSR_SURV_CSTRIDE], (uint32_t)__popcll(mk));
            at = (uint32_t)__builtin_amdgcn_readfirstlane((int)at);
            if (surv) a.surv.ids[(size_t)sl * a.surv.cap + at + (uint32_t)__popcll(mk & ((1ull << lane) - 1ull))] = (uint32_t)idx;
        }
    }
    if (a.dirty != nullptr && live && !surv && !a.guard.frozen()) {
        const uint8_t d = a.dirty[idx];
        if (d != 0) { zero_grad_rows(a.rows, (size_t)idx, (d & 1) != 0, (d & 2) != 0); a.dirty[idx] = 0; }
    }
#if GSR_TIMING
    const long long tp3_ = clock64();
#endif
    // k_preprocess_lean (a.sh_here): the wave's lanes are dense with survivors, so their colour is evaluated right here -- one
    // kernel (and one chain of dependent memory phases) less per iteration than with k_sh_color behind this one.
    if (FLAT && a.sh_here) asm volatile("" : : "v"(sh_touch0), "v"(sh_touch1));      // (keeps the two touches above alive up to here)
    if (FLAT && a.sh_here && surv) {
        uint8_t cb;
        const float3 c = sh16_vector_ok(a.M, a.shs)
                             ? sh_row16_to_rgb(a.D, p, a.campos, reinterpret_cast<const float4*>(a.shs) + (size_t)idx * GSR_SH16_ROW4, cb)
                             : sh_to_rgb(a.D, a.M, p, a.campos, a.shs + (size_t)idx * a.M * 3, cb);
        reinterpret_cast<float4*>(a.rec + (size_t)idx * GSR_REC_STRIDE)[2] = make_float4(c.x, c.y, c.z, 0.f);
        a.clamped[idx] = cb;
    }
#if GSR_TIMING
    if (FLAT && s_flat != nullptr && (tid & 63) == 0) {
        const long long tp4_ = clock64();
        s_flat[129] += (uint32_t)(tp1_ - tp0_); s_flat[130] += (uint32_t)(tp2_ - tp1_); s_flat[131] += (uint32_t)(tp3_ - tp2_); s_flat[132] += (uint32_t)(tp4_ - tp3_);
    }
#endif
}

__global__ void __launch_bounds__(GSR_BLOCK) k_preprocess(PreArgs a)
{
    // (the per-tile bounds are read straight from global memory: only the few lanes of a wave whose splat survives
    // the superblock test look at them, a dozen reads per wave that hit in L1/L2, against 1 200 loads + LDS stores and
    // a barrier per workgroup for a staged copy -- an eighth of the kernel's time, and a limit on the tile count)
    extern __shared__ float s_zbc[];      // a.zbc_lds floats: the superblock bounds (0: read them from global memory)
    const int tid = threadIdx.x;
    if (a.tile_order[0] != nullptr && blockIdx.x < 2) {      // (before the poison test: the orders must be permutations whatever happens)
        __shared__ uint32_t s_cls[GSR_BLOCK];
        tile_order_from_work(a.tile_work[blockIdx.x], a.tile_order[blockIdx.x], a.order_tiles, s_cls);
    }
    if (a.guard.poisoned()) return;
    GSR_T_DECL
    if (a.zbc_lds > 0) {
        const float* bsrc = a.pyr_tiles ? a.zb : a.zbc;
        for (int i = tid; i < a.zbc_lds; i += GSR_BLOCK) s_zbc[i] = bsrc[i];
        __syncthreads();
        build_bound_pyramid(s_zbc, a.pyr_tiles ? a.gx : a.sbx, a.pyr_tiles ? a.gy : a.sby);
    }
    const int idx = blockIdx.x * GSR_BLOCK + tid;
    if (a.tile_count != nullptr && idx < a.ntiles) a.tile_count[idx] = 0u;      // (k_tile_count adds into them next)
    if (idx == 0) {      // the null splat
        float4* nr = reinterpret_cast<float4*>(a.rec + (size_t)a.P * GSR_REC_STRIDE);
        nr[0] = make_float4(0.f, 0.f, 0.f, 0.f); nr[1] = nr[0]; nr[2] = nr[0];
    }
    preprocess_one<false>(a, idx, idx < a.P, s_zbc, tid, blockIdx.x & (GSR_SURV_LISTS - 1));
}

// ---------------------------------------------------------------------------------------------
// The preprocess of a native-loop iteration whose `radii` the caller cannot get (PreArgs::lean: speculative binning, not
// the last iteration).  98 % of the Gaussians in front of the camera lie behind the depth bound of every tile they could
// touch and would leave k_preprocess with tiles_touched = 0 -- after ~1 000 instructions of exact geometry and footprint walk,
// which a wave executes in full as soon as ONE of its 64 lanes needs it (two waves out of three on S-1M-640, for 1.7 lanes).
// Here a wave looks at GSR_LEAN_PER_LANE x 64 Gaussians:
//   1. every lane bounds its Gaussians' radii from a stored bound on their 3D extent (PreArgs::lam, lean_candidate):
//         lambda_max(cov2D + 0.3 I) <= |J|_F^2 |W|_2^2 lambda_max(Sigma) + 0.3
//      which gives a rectangle that contains the exact one; behind the bounds of all ITS superblocks => behind every tile's:
//      settled, and nothing is written for such a Gaussian (neither radii nor tiles_touched are read in such an iteration:
//      the consumers walk the survivor lists);
//   2. the others -- under 2 %, four or five per wave -- are compacted (ballot + prefix, the wave's own 1 KB of LDS, no workgroup
//      barrier) and the wave runs preprocess_one ONCE on them, dense lanes, flattened footprint walk.
// A frozen (converged) iteration's forward is the render the caller gets back, radii included: then nobody is settled, the
// flags are zeroed here, and the kernel computes exactly what k_preprocess would.
// ---------------------------------------------------------------------------------------------
#ifndef GSR_LEAN_OCC
#define GSR_LEAN_OCC 4      // waves per SIMD the register allocation aims at (experiments: -DGSR_LEAN_OCC=5 -> 93 VGPRs + 12 B of scratch)
#endif
__global__ void __launch_bounds__(GSR_BLOCK, GSR_LEAN_OCC) k_preprocess_lean(PreArgs a)
{
    extern __shared__ float s_zbc[];      // a.zbc_lds floats: the superblock bounds
    __shared__ uint32_t s_cand[4][GSR_LEAN_PER_LANE * 64];
    __shared__ uint32_t s_flat[4][136];      // (128 words per wave; words 128-133: diagnostics of the timing build)
    const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
    if (a.tile_order[0] != nullptr && blockIdx.x < 2) {      // (before the poison test: the orders must be permutations whatever happens)
        __shared__ uint32_t s_cls[GSR_BLOCK];
        tile_order_from_work(a.tile_work[blockIdx.x], a.tile_order[blockIdx.x], a.order_tiles, s_cls);
    }
    if (a.guard.poisoned()) return;
    GSR_T_DECL
    {
        const float* bsrc = a.pyr_tiles ? a.zb : a.zbc;
        for (int i = tid; i < a.zbc_lds; i += GSR_BLOCK) s_zbc[i] = bsrc[i];
    }
    __syncthreads();
    build_bound_pyramid(s_zbc, a.pyr_tiles ? a.gx : a.sbx, a.pyr_tiles ? a.gy : a.sby);
    GSR_T_TICK(0)
    const bool frozen = a.guard.frozen();
    if (blockIdx.x == 0 && tid == 0) {      // the null splat
        float4* nr = reinterpret_cast<float4*>(a.rec + (size_t)a.P * GSR_REC_STRIDE);
        nr[0] = make_float4(0.f, 0.f, 0.f, 0.f); nr[1] = nr[0]; nr[2] = nr[0];
    }
    // Which Gaussians a wave looks at: not 256 consecutive ones but sixteen SEGMENTS of sixteen, taken round-robin over all waves
    // (segment s belongs to wave s mod #waves; a load instruction still moves four 256-byte runs).  Maps come in whatever order
    // their training left them in -- spatially correlated, a Morton-sorted one in the extreme -- and the candidates of an iteration
    // (the front layer of the scene) then sit in a few long index runs: with consecutive ranges the waves owning those runs went
    // through the exact pass four times over while the others had nothing (k_preprocess_lean 164 instead of 34 us on a sorted
    // S-1M-640, 289 instead of 60 on S-3M-cam; now 45 and 68).  Round-robin segments hand every wave the same share of every run.
    // (round-robin inside windows of GSR_LEAN_WINDOW waves = 64 K Gaussians: over the whole map it costs the 16-byte stream its
    // locality -- 64.6 instead of 60.0 us at 3 M Gaussians in random order)
#ifndef GSR_LEAN_INTERLEAVE
#define GSR_LEAN_INTERLEAVE 1
#endif
    const int wave_global = blockIdx.x * 4 + wv;
    auto idx_of = [&](int k) {
        return GSR_LEAN_INTERLEAVE ? ((wave_global / GSR_LEAN_WINDOW) * (GSR_LEAN_WINDOW * GSR_LEAN_PER_LANE * 64) +
                                      ((4 * k + (lane >> 4)) * GSR_LEAN_WINDOW + (wave_global % GSR_LEAN_WINDOW)) * 16 + (lane & 15))
                                   : (wave_global * (GSR_LEAN_PER_LANE * 64) + k * 64 + lane);
    };
    int ncand = 0;                             // wave-uniform
    // (all the loads of the wave's Gaussians first: one round trip, not one per sub-chunk)
    float3 pk[GSR_LEAN_PER_LANE]; float sk[GSR_LEAN_PER_LANE]; uint8_t dk[GSR_LEAN_PER_LANE];
#pragma unroll
    for (int k = 0; k < GSR_LEAN_PER_LANE; k++) {
        const int idx = min(idx_of(k), a.P - 1);
        const float4 ml = reinterpret_cast<const float4*>(a.lam)[idx];      // (mean, extent bound): one coalesced 16-byte load
        pk[k] = make_float3(ml.x, ml.y, ml.z);
        sk[k] = ml.w;
        dk[k] = (a.dirty != nullptr) ? a.dirty[idx] : (uint8_t)0;
    }
    const float wn2 = view_norm2_bound(a.view);
#pragma unroll
    for (int k = 0; k < GSR_LEAN_PER_LANE; k++) {
        const int idx = idx_of(k);
        const bool live = idx < a.P;
        bool cand = false;
        if (live) {
            if (frozen) { a.radii[idx] = 0; a.tiles_touched[idx] = 0; }
            const float3 p = pk[k];
            const float3 pview = xform4x3(p, a.view);
            if (pview.z > 0.2f)       // near cull (auxiliary.h:150); a frozen forward's radii are an output: nobody is settled
                cand = frozen ? true : lean_candidate<true>(a, p, pview, sk[k], wn2, s_zbc);
        }
        // (a Gaussian that is not even a candidate gets no gradient this iteration: see PreArgs::dirty; candidates: preprocess_one)
        if (a.dirty != nullptr && live && !cand && !frozen) {
            const uint8_t d = dk[k];
            if (d != 0) { zero_grad_rows(a.rows, (size_t)idx, (d & 1) != 0, (d & 2) != 0); a.dirty[idx] = 0; }
        }
        const unsigned long long mk = __ballot(cand);
        if (cand) s_cand[wv][ncand + (int)__popcll(mk & ((1ull << lane) - 1ull))] = (uint32_t)idx;
        ncand += (int)__popcll(mk);
    }
    __builtin_amdgcn_wave_barrier();
    GSR_T_TICK(1)
    GSR_T_COUNT(10, ncand)
#if GSR_TIMING
    if (lane == 0) { s_flat[wv][128] = 0u; s_flat[wv][129] = 0u; s_flat[wv][130] = 0u; s_flat[wv][131] = 0u; s_flat[wv][132] = 0u; s_flat[wv][133] = 0u; s_flat[wv][134] = 0u; }
    __builtin_amdgcn_wave_barrier();
#endif
#if GSR_LEAN_POOL > 1
    // The exact pass costs ~1 800 vector instructions per WAVE whether four of its lanes are live or sixty-four: GSR_LEAN_POOL
    // neighbouring waves hand their candidates to the first of them (the conservative passes end within a few hundred cycles of each
    // other since the bound pyramid), which runs ONE exact pass on the pooled list; the others are done.
    __shared__ int s_ncand[4];
    if (lane == 0) s_ncand[wv] = ncand;
    __syncthreads();
    if ((wv % GSR_LEAN_POOL) != 0) { GSR_T_TICK(2) GSR_T_FLUSH(32) return; }
    int pooled = 0;
#pragma unroll
    for (int w = 0; w < GSR_LEAN_POOL; w++) pooled += s_ncand[wv + w];
    for (int c0 = 0; c0 < pooled; c0 += 64) {
        const int j = c0 + lane;
        const bool mine = j < pooled;
        int idx = 0, run = 0;
#pragma unroll
        for (int w = 0; w < GSR_LEAN_POOL; w++) {          // (candidate j of the pooled list: wave w's list behind wave w - 1's)
            const int n_w = s_ncand[wv + w];
            if (mine && j >= run && j < run + n_w) idx = (int)s_cand[wv + w][j - run];
            run += n_w;
        }
        preprocess_one<true>(a, idx, mine, s_zbc, tid, blockIdx.x & (GSR_SURV_LISTS - 1), s_flat[wv]);
    }
#else
    for (int c0 = 0; c0 < ncand; c0 += 64) {
        const bool mine = c0 + lane < ncand;
        preprocess_one<true>(a, mine ? (int)s_cand[wv][c0 + lane] : 0, mine, s_zbc, tid, blockIdx.x & (GSR_SURV_LISTS - 1), s_flat[wv]);
    }
#endif
    GSR_T_TICK(2)
#if GSR_TIMING
    __builtin_amdgcn_wave_barrier();
    GSR_T_COUNT(11, s_flat[wv][128])
    // (sub-phases of the exact passes, summed over them: slots 3-6 = geometry incl. the hoisted loads | footprint walk + appends |
    // survivors' list + dirty rows | SH colour)
    GSR_T_COUNT(3, s_flat[wv][129]) GSR_T_COUNT(4, s_flat[wv][130]) GSR_T_COUNT(5, s_flat[wv][131]) GSR_T_COUNT(6, s_flat[wv][132])
    GSR_T_COUNT(7, s_flat[wv][133]) GSR_T_COUNT(8, s_flat[wv][134])
#endif
    GSR_T_FLUSH(32)
}

// Differential check of the conservative test (gsr_debug_lean_check; tests only).  One lane per Gaussian: lean_candidate with
// the same inputs k_preprocess_lean gives it, and next to it the exact geometry of preprocess_one (same building blocks, same
// expression order) with the exact footprint walk against the same per-tile bounds, counting instead of appending.
// out[0] settled, out[1] candidates, out[2] Gaussians the exact walk bins somewhere, out[3] settled AND binned (violations),
// out[4] smallest violating index + 1 (atomicMin on ~index is awkward: kept as max of ~idx).
__global__ void __launch_bounds__(GSR_BLOCK) k_lean_check(PreArgs a, unsigned long long* out)
{
    const int idx = blockIdx.x * GSR_BLOCK + threadIdx.x;
    if (idx >= a.P) return;
    const float3 p = make_float3(a.means[3 * idx], a.means[3 * idx + 1], a.means[3 * idx + 2]);
    const float3 pview = xform4x3(p, a.view);
    bool cand = false;
    uint32_t cnt = 0;
    if (pview.z > 0.2f) {
        // (the bounds without the coarser levels k_preprocess_lean adds in LDS -- the exact maximum over the rectangle's tiles, or over its
        // superblocks where the kernel starts from those: what this settles is a superset of what the kernel settles)
        cand = lean_candidate<false>(a, p, pview, a.lam[4 * (size_t)idx + 3], view_norm2_bound(a.view), a.pyr_tiles ? a.zb : a.zbc);
        const float4 ph = xform4x4(p, a.proj);
        const float pw = 1.0f / (ph.w + 0.0000001f);
        const float3 pproj = make_float3(ph.x * pw, ph.y * pw, ph.z * pw);
        float cov6[6];
#pragma unroll
        for (int i = 0; i < 6; i++) cov6[i] = a.cov3D_pre[6 * (size_t)idx + i];
        Cov2DTerms ct;
        cov2d_terms(p, a.fx, a.fy, a.tanx, a.tany, cov6, a.view, ct);
        const float cx = ct.cov.m[0][0] + 0.3f, cy = ct.cov.m[0][1], cz = ct.cov.m[1][1] + 0.3f;
        const float det = (cx * cz - cy * cy);
        if (det != 0.0f) {
            const float det_inv = 1.f / det;
            const float3 conic = make_float3(cz * det_inv, -cy * det_inv, cx * det_inv);
            const float mid = 0.5f * (cx + cz);
            const float lambda1 = mid + sqrtf(fmaxf(0.1f, mid * mid - det));
            const float lambda2 = mid - sqrtf(fmaxf(0.1f, mid * mid - det));
            const float my_radius = ceilf(3.f * sqrtf(fmaxf(lambda1, lambda2)));
            const float2 pix = make_float2(ndc2pix(pproj.x, a.W), ndc2pix(pproj.y, a.H));
            int x0, y0, x1, y1;
            get_rect(pix.x, pix.y, (int)my_radius, a.gx, a.gy, x0, y0, x1, y1);
            if ((x1 - x0) * (y1 - y0) != 0) {
                const TileTest tt = make_tile_test(pix, conic, a.opac[idx]);
                clip_rect(tt, x0, y0, x1, y1);
                for (int y = y0; y < y1; y++) {
                    int lo, hi;
                    row_span(tt, y, x0, x1, lo, hi);
                    for (int x = lo; x <= hi; x++)
                        if (pview.z <= a.zb[y * a.gx + x] * a.zb_mul + a.zb_add) cnt++;
                }
            }
        }
    }
    const bool bad = !cand && cnt != 0u;
    const unsigned long long m_set = __ballot(!cand), m_cand = __ballot(cand), m_bin = __ballot(cnt != 0u), m_bad = __ballot(bad);
    if ((threadIdx.x & 63) == 0) {
        atomicAdd(&out[0], (unsigned long long)__popcll(m_set));
        atomicAdd(&out[1], (unsigned long long)__popcll(m_cand));
        atomicAdd(&out[2], (unsigned long long)__popcll(m_bin));
        if (m_bad != 0ull) atomicAdd(&out[3], (unsigned long long)__popcll(m_bad));
    }
    if (bad) atomicMax(&out[4], (unsigned long long)(0xFFFFFFFFu - (uint32_t)idx));      // -> smallest violating index
}

// SH -> RGB (forward.cu:20-71) as its own kernel: it only needs the survivors of the geometry pass, so the host
// runs it on a side stream underneath the (latency-bound) binning chain and joins before compositing.
// Summation order is the reference's.
#define GSR_SHC_ROWS 64
// One WAVE per 64-entry chunk of a work list (workgroup w: sub-list w mod GSR_SURV_LISTS, chunks w / GSR_SURV_LISTS, ... in
// steps of gridDim / GSR_SURV_LISTS): the chunk's 192-B SH rows are staged through LDS as 16-B-per-lane streams and every
// lane then evaluates one Gaussian.  The kernel is a chain of dependent memory phases per wave (list -> rows -> stores), so
// the host launches at most as many waves as are resident at once (129 registers, 13 KB of LDS: 8 per CU).
#define GSR_SHC_RESIDENT (256 * 8)
__global__ void __launch_bounds__(64) k_sh_color(PreArgs a)
{
    __shared__ float4 s_sh[GSR_SHC_ROWS * GSR_SH16_LDS4];
    const int lane = threadIdx.x;
    if (a.guard.poisoned()) return;
    // only splats that were binned into at least one tile can ever be composited (this also skips everything
    // the native loop's speculative depth bounds dropped)
    const uint32_t sl = blockIdx.x & (GSR_SURV_LISTS - 1);
    const uint32_t n = a.surv.n[sl * GSR_SURV_CSTRIDE];
    const uint32_t* __restrict__ list = a.surv.ids + (size_t)sl * a.surv.cap;
    const uint32_t step = (gridDim.x / GSR_SURV_LISTS) * GSR_SHC_ROWS;
    const bool staged = sh16_vector_ok(a.M, a.shs);
    for (uint32_t c0 = (blockIdx.x / GSR_SURV_LISTS) * GSR_SHC_ROWS; c0 < n; c0 += step) {
        const int nrow = (int)min((uint32_t)GSR_SHC_ROWS, n - c0);
        const int idx = (lane < nrow) ? (int)list[c0 + lane] : 0;
        if (staged) {
#pragma unroll
            for (int i = 0; i < GSR_SH16_ROW4; i++) {
                const int j = lane + 64 * i;
                const int r = j / GSR_SH16_ROW4, part = j - r * GSR_SH16_ROW4;
                const int rid = __shfl(idx, r, 64);
                if (r < nrow) s_sh[r * GSR_SH16_LDS4 + part] = reinterpret_cast<const float4*>(a.shs)[(size_t)rid * GSR_SH16_ROW4 + part];
            }
        }
        __syncthreads();
        if (lane < nrow) {
            const float3 p = make_float3(a.means[3 * idx], a.means[3 * idx + 1], a.means[3 * idx + 2]);
            uint8_t cb;
            const float3 c = staged ? sh_to_rgb(a.D, 16, p, a.campos, reinterpret_cast<const float*>(&s_sh[lane * GSR_SH16_LDS4]), cb)
                                    : sh_to_rgb(a.D, a.M, p, a.campos, a.shs + (size_t)idx * a.M * 3, cb);
            reinterpret_cast<float4*>(a.rec + (size_t)idx * GSR_REC_STRIDE)[2] = make_float4(c.x, c.y, c.z, 0.f);
            a.clamped[idx] = cb;
        }
        __syncthreads();
    }
}

// ---------------------------------------------------------------------------------------------
// Binning with complete lists ("exact bins"; every forward that has no depth bounds to speculate with).
// The reference duplicates every Gaussian into R (tile<<32 | depth) keys and radix-sorts all of them
// (rasterizer_impl.cu:70-111, 278-315: 6 passes over R pairs).  95 % of that sorted list is never looked at: a tile's
// pixels saturate after the first few hundred entries.  Here nothing is sorted globally:
//   k_tile_count   every (Gaussian, tile) pair that survives the exact ellipse test is counted per tile -- in LDS, per
//                  workgroup of a few thousand Gaussians, so that the tile counters in HBM see one add per
//                  (workgroup, tile) instead of one per instance (memory-side atomics: ~18 per ns);
//   k_tile_scan    exclusive prefix sum over the tile counts = every tile's segment of the instance arrays (and the
//                  total, which the host reads to size them: the reference's one blocking read, rasterizer_impl.cu:282);
//   k_tile_emit    the same walk again: a workgroup reserves its share of each tile's segment with one returning atomic
//                  per (workgroup, tile) and scatters its (depth bits << 32 | index) keys there, in no particular order;
//   compositing    k_render_fwd<.., 2> orders a tile's segment lazily, front to back: it SELECTS the nearest couple of
//                  hundred keys (a depth threshold from a sample, one gather pass: sample_slice), sorts those (in registers
//                  up to 256, bitonic in LDS above), composites them, and only goes back for the next slice while some pixel
//                  of the tile is still unsaturated.
// The order inside a tile is (depth bits, index) -- what the reference's stable sort of (tile | depth) keys gives -- as
// far as the walk gets; the sorted prefix is written out for the backward pass, which never reads beyond the deepest
// contributor.
// ---------------------------------------------------------------------------------------------
#define GSR_TBIN_COOP 32          // rectangles with more tiles than this are walked by the whole wave
// Every workgroup adds its per-tile counts into the tile counters in HBM; with all of them hammering the same few KB the
// memory-side atomic unit serialises (MI355X_MICROARCH.md, "Global float atomics": everybody into one row = 14x slower).
// The counters are therefore kept in GSR_TBIN_COPIES private copies (workgroup b uses copy b mod copies); k_tile_scan adds
// the copies up and gives every copy its own sub-range of the tile's segment.
#ifndef GSR_TBIN_COPIES
#define GSR_TBIN_COPIES 4          // (1: emit +10 %; 16: the single-workgroup scan takes 20-40 us; measured on S-1M-640 and the 1.5 M training scene)
#endif
// Workgroups of 1024 lanes: the walk is a short chain of dependent loads per Gaussian, so what counts is how many of them
// are in flight -- 16 waves per workgroup, two workgroups per CU -- while the LDS counters still aggregate a few thousand
// Gaussians.
#define GSR_TBIN_THREADS 1024
#ifndef GSR_RESERVE_ROT
#define GSR_RESERVE_ROT 67u      // workgroup b starts its reservation atomics at tile (b x this) mod ntiles (0: everybody at tile 0)
#endif
struct TileBinArgs {
    int P, gx, gy, ntiles, gpb;                    // gpb: Gaussians per workgroup (multiple of GSR_TBIN_THREADS)
    int copies;                                    // private copies of the per-tile counters (1 ... GSR_TBIN_COPIES)
    const uint32_t* tiles_touched; const ushort4* rects; const float* rec;
    uint32_t* tile_count;                          // [copies][ntiles]: the count kernel adds into them
    const uint32_t* tile_start;                    // [copies][ntiles]: start of each copy's sub-range inside the tile's segment (scan -> emit)
    const uint32_t* tile_offset;                   // [ntiles + 1]   (emit)
    uint32_t* tile_fill;                           // [copies][ntiles]: how much of each sub-range has been handed out (emit)
    uint16_t* block_counts;                        // [workgroups][ntiles]: what each workgroup counted (count writes, emit reads); LDSAGG only
    unsigned long long* keys;                      // [R] (emit)
};

// (g0: offset of the KPT x 1024 window inside the workgroup's gpb Gaussians)
template <int KPT>
__device__ __forceinline__ void walk_load(const TileBinArgs& a, int g0, WalkItem (&it)[KPT])
{
    const int base = blockIdx.x * a.gpb + g0;
#pragma unroll
    for (int k = 0; k < KPT; k++) {
        const int idx = base + k * GSR_TBIN_THREADS + (int)threadIdx.x;
        WalkItem w = {};
        if (g0 + k * GSR_TBIN_THREADS < a.gpb && idx < a.P && a.tiles_touched[idx] != 0u) {
            const ushort4 r = a.rects[idx];
            const SplatRec sr = load_splat_rec(a.rec, (uint32_t)idx);
            const TileTest tt = make_tile_test(make_float2(sr.x, sr.y), make_float3(sr.a, sr.b, sr.c), sr.opacity);
            w.x0 = r.x; w.y0 = r.y; w.x1 = r.z; w.y1 = r.w;
            clip_rect(tt, w.x0, w.y0, w.x1, w.y1);
            w.mx = tt.mx; w.my = tt.my; w.at = tt.A * tt.twoq; w.B = tt.B; w.det = tt.det; w.dye = tt.dye; w.invA = tt.invA;
            w.all = !tt.cull;
            w.key = ((unsigned long long)__float_as_uint(sr.depth) << 32) | (uint32_t)idx;
        }
        it[k] = w;
    }
}
// Calls visit(tile, key) for every tile instance of the cached Gaussians in tile rows [b0, b1).
// Footprints differ by two orders of magnitude (1 ... hundreds of tiles), so the unit of work handed to a lane is not a
// Gaussian but one ROW of one Gaussian's rectangle: the wave lays the rows of its 64 Gaussians end to end (prefix sum of
// the row counts), takes them 64 at a time, and each lane looks up whose row it got (binary search in the wave's prefix
// array, in LDS), fetches that Gaussian's span terms from the owning lane (ds_bpermute) and walks the row's span.
// s_pref: 64 words of LDS per wave.
template <int KPT, class Visit>
__device__ __forceinline__ void walk_rows(const TileBinArgs& a, const WalkItem (&it)[KPT], int b0, int b1, uint32_t* s_pref, Visit&& visit)
{
    const int lane = threadIdx.x & 63;
    uint32_t* pref = s_pref + (threadIdx.x >> 6) * 64;
#define GSR_PERM_F(v, src) __uint_as_float((uint32_t)__builtin_amdgcn_ds_bpermute((src) << 2, (int)__float_as_uint(v)))
#define GSR_PERM_I(v, src) __builtin_amdgcn_ds_bpermute((src) << 2, (int)(v))
#pragma unroll
    for (int k = 0; k < KPT; k++) {
        const WalkItem& w = it[k];
        const int y0 = max(w.y0, b0), y1 = min(w.y1, b1);
        const int nrows = (w.x1 > w.x0 && y1 > y0) ? (y1 - y0) : 0;
        int incl = nrows;
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
            const int o = __shfl_up(incl, off, 64);
            if (lane >= off) incl += o;
        }
        const int total = __builtin_amdgcn_readlane(incl, 63);
        if (total == 0) continue;                  // wave-uniform
        pref[lane] = (uint32_t)(incl - nrows);     // first row slot of lane's Gaussian (same-wave LDS traffic is in order: no barrier)
        __builtin_amdgcn_wave_barrier();
        for (int p0 = 0; p0 < total; p0 += 64) {
            const int p = p0 + lane;
            const bool act = p < total;
            int src = 0;
            if (act) {                             // largest lane s with pref[s] <= p (lanes with no rows share their successor's start:
#pragma unroll                                     //  the largest one is the owner)
                for (int step = 32; step > 0; step >>= 1)
                    if (pref[src + step] <= (uint32_t)p) src += step;
            }
            WalkItem r;
            r.mx = GSR_PERM_F(w.mx, src); r.my = GSR_PERM_F(w.my, src); r.at = GSR_PERM_F(w.at, src); r.B = GSR_PERM_F(w.B, src);
            r.det = GSR_PERM_F(w.det, src); r.dye = GSR_PERM_F(w.dye, src); r.invA = GSR_PERM_F(w.invA, src);
            r.x0 = GSR_PERM_I(w.x0, src); r.x1 = GSR_PERM_I(w.x1, src);
            r.all = GSR_PERM_I((int)w.all, src) != 0;
            const uint32_t klo = (uint32_t)GSR_PERM_I((uint32_t)w.key, src), khi = (uint32_t)GSR_PERM_I((uint32_t)(w.key >> 32), src);
            const int sy0 = GSR_PERM_I(y0, src);
            const int sfirst = GSR_PERM_I(incl - nrows, src);
            if (act) {
                const unsigned long long key = ((unsigned long long)khi << 32) | klo;
                const int y = sy0 + (p - sfirst);
                int lo, hi;
                item_span(r, y, lo, hi);
                for (int x = lo; x <= hi; x++) visit(y * a.gx + x, key);
            }
        }
    }
#undef GSR_PERM_F
#undef GSR_PERM_I
}

// LDSAGG: the workgroup's per-tile counters live in LDS (a.ntiles words of dynamic shared memory); false: images with more
// tiles than LDS can hold counters for, or more Gaussians per workgroup than KPT x 1024 -- every instance adds to the
// counters in HBM directly (one copy).
template <bool LDSAGG, int KPT>
__global__ void __launch_bounds__(GSR_TBIN_THREADS) k_tile_count(TileBinArgs a)
{
    extern __shared__ uint32_t s_tb[];
    __shared__ uint32_t s_pref[GSR_TBIN_THREADS];
    WalkItem it[KPT];
    if (LDSAGG) {
        for (int t = threadIdx.x; t < a.ntiles; t += GSR_TBIN_THREADS) s_tb[t] = 0u;
        walk_load<KPT>(a, 0, it);
        __syncthreads();
        walk_rows<KPT>(a, it, 0, a.gy, s_pref, [&](int tile, unsigned long long) { atomicAdd(&s_tb[tile], 1u); });
        __syncthreads();
        uint32_t* mine = a.tile_count + (size_t)(blockIdx.x % a.copies) * a.ntiles;
        uint16_t* row = a.block_counts + (size_t)blockIdx.x * a.ntiles;
        for (int t = threadIdx.x; t < a.ntiles; t += GSR_TBIN_THREADS) {      // consecutive lanes -> consecutive counters: 256-B atomic bursts
            const uint32_t c = s_tb[t];
            row[t] = (uint16_t)c;                                      // (at most one instance per Gaussian and tile: c <= gpb <= 8192)
            if (c != 0u) atomicAdd(&mine[t], c);
        }
    } else {
        for (int g0 = 0; g0 < a.gpb; g0 += KPT * GSR_TBIN_THREADS) {
            WalkItem jt[KPT];
            walk_load<KPT>(a, g0, jt);
            walk_rows<KPT>(a, jt, 0, a.gy, s_pref, [&](int tile, unsigned long long) { atomicAdd(&a.tile_count[tile], 1u); });
        }
    }
}

// One workgroup.  Per tile: total over the counter copies; tile_offset = exclusive prefix sum of the totals (ntiles + 1
// entries); tile_start[copy][tile] = where that copy's sub-range begins inside the tile's segment; tile_fill = 0;
// the grand total goes to *total_out and, if given, to a word of pinned host memory the host is polling (host_total[0] =
// total, host_total[1] = seq, written last).  Each lane owns a run of consecutive tiles: one round of independent loads,
// one block-wide scan of the per-lane sums, one round of stores.
#define GSR_TSCAN_PER_LANE 16          // 1024 lanes x 16 tiles: up to 16 384 tiles per pass (more: passes with a carry)
__global__ void __launch_bounds__(1024) k_tile_scan(int ntiles, int copies, const uint32_t* __restrict__ tile_count, uint32_t* __restrict__ tile_start,
                                                     uint32_t* __restrict__ tile_offset, uint32_t* __restrict__ tile_fill,
                                                     uint32_t* __restrict__ total_out, volatile uint32_t* host_total, uint32_t seq)
{
    __shared__ uint32_t s_wave[16];
    __shared__ uint32_t s_carry;
    const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
    if (tid == 0) s_carry = 0u;
    __syncthreads();
    const int per = min(GSR_TSCAN_PER_LANE, (ntiles + 1023) / 1024);
    for (int t0 = 0; t0 < ntiles; t0 += 1024 * per) {
        const int first = t0 + tid * per;
        uint32_t tot[GSR_TSCAN_PER_LANE];
        uint32_t mine = 0u;
#pragma unroll
        for (int q = 0; q < GSR_TSCAN_PER_LANE; q++) {
            tot[q] = 0u;
            const int t = first + q;
            if (q < per && t < ntiles) {
                uint32_t v[GSR_TBIN_COPIES];              // all copies first: independent loads, one round trip
#pragma unroll
                for (int k = 0; k < GSR_TBIN_COPIES; k++) v[k] = (k < copies) ? tile_count[(size_t)k * ntiles + t] : 0u;
                uint32_t c = 0u;
#pragma unroll
                for (int k = 0; k < GSR_TBIN_COPIES; k++)
                    if (k < copies) {
                        tile_start[(size_t)k * ntiles + t] = c;          // start of copy k's sub-range, relative to the tile's segment
                        tile_fill[(size_t)k * ntiles + t] = 0u;
                        c += v[k];
                    }
                tot[q] = c;
                mine += c;
            }
        }
        uint32_t incl = mine;
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
            const uint32_t o = __shfl_up(incl, off, 64);
            if (lane >= off) incl += o;
        }
        if (lane == 63) s_wave[wv] = incl;
        __syncthreads();
        uint32_t run = s_carry + incl - mine;
        for (int w = 0; w < wv; w++) run += s_wave[w];
#pragma unroll
        for (int q = 0; q < GSR_TSCAN_PER_LANE; q++) {
            const int t = first + q;
            if (q < per && t < ntiles) { tile_offset[t] = run; run += tot[q]; }
        }
        __syncthreads();
        if (tid == 1023) s_carry = run;
        __syncthreads();
    }
    if (tid == 0) {
        tile_offset[ntiles] = s_carry;
        *total_out = s_carry;
        if (host_total != nullptr) { host_total[0] = s_carry; __threadfence_system(); host_total[1] = seq; }
    }
}

// The emit makes `bands` passes over the image, a band of tile rows at a time: every workgroup writes its keys of band 0,
// then of band 1, ...  All workgroups are resident and move at about the same pace, so at any moment the scattered 8-byte
// stores of the whole chip fall into one band's share of the key array -- small enough to sit in the L2s until its 64-byte
// lines are complete (measured without bands at 1.5 M Gaussians / 4 293 tiles: 230-610 MB written for 96 MB of keys).
// The per-Gaussian terms are computed once and kept in registers across the passes.
template <bool LDSAGG, int KPT>
__global__ void __launch_bounds__(GSR_TBIN_THREADS) k_tile_emit(TileBinArgs a, int bands)
{
    extern __shared__ uint32_t s_tb[];        // LDSAGG: [0, ntiles) running count, [ntiles, 2 ntiles) where this workgroup's keys of the tile start
    __shared__ uint32_t s_pref[GSR_TBIN_THREADS];
    if (LDSAGG) {
        uint32_t* s_cnt = s_tb;
        uint32_t* s_base = s_tb + a.ntiles;
        const size_t copy = (size_t)(blockIdx.x % a.copies) * a.ntiles;
        const uint16_t* row = a.block_counts + (size_t)blockIdx.x * a.ntiles;
        // (four returning atomics in flight per lane, every workgroup starting at another tile: see k_preprocess_bin)
        const int rot = (int)((blockIdx.x * GSR_RESERVE_ROT) % (uint32_t)a.ntiles);
        for (int t0 = threadIdx.x; t0 < a.ntiles; t0 += 4 * GSR_TBIN_THREADS) {
            int tt[4];
            uint32_t c[4], b[4];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const int t = t0 + j * GSR_TBIN_THREADS;
                tt[j] = (t < a.ntiles) ? ((t + rot >= a.ntiles) ? t + rot - a.ntiles : t + rot) : -1;
                c[j] = (tt[j] >= 0) ? row[tt[j]] : 0u;          // what this workgroup counted for the tile (k_tile_count): reserve that much
            }
#pragma unroll
            for (int j = 0; j < 4; j++)
                b[j] = (c[j] != 0u) ? a.tile_offset[tt[j]] + a.tile_start[copy + tt[j]] + atomicAdd(&a.tile_fill[copy + tt[j]], c[j]) : 0u;
#pragma unroll
            for (int j = 0; j < 4; j++)
                if (tt[j] >= 0) { s_base[tt[j]] = b[j]; s_cnt[tt[j]] = 0u; }
        }
        WalkItem it[KPT];
        walk_load<KPT>(a, 0, it);
        const int bh = (a.gy + bands - 1) / bands;
        for (int b0 = 0; b0 < a.gy; b0 += bh) {
            __syncthreads();
            walk_rows<KPT>(a, it, b0, min(a.gy, b0 + bh), s_pref,
                           [&](int tile, unsigned long long key) { a.keys[s_base[tile] + atomicAdd(&s_cnt[tile], 1u)] = key; });
        }
    } else {
        for (int g0 = 0; g0 < a.gpb; g0 += KPT * GSR_TBIN_THREADS) {
            WalkItem jt[KPT];
            walk_load<KPT>(a, g0, jt);
            walk_rows<KPT>(a, jt, 0, a.gy, s_pref,
                           [&](int tile, unsigned long long key) { a.keys[a.tile_offset[tile] + atomicAdd(&a.tile_fill[tile], 1u)] = key; });
        }
    }
}

// ---------------------------------------------------------------------------------------------
// Complete lists in ONE kernel (round 3): preprocess + count + reserve + emit.  k_preprocess -> k_tile_count -> k_tile_scan ->
// [host reads the total] -> k_tile_emit moved every visible Gaussian's record through HBM twice more (both walks re-read it and
// re-derived the span terms: 299 MB per forward on S-1M-640 for 148 MB of algorithmic traffic), needed a single-workgroup scan in
// the middle and a blocking read to size the key array.  Here a workgroup of 1024 lanes computes the geometry of its KPT x 1024
// Gaussians (preprocess_one, the same code), keeps each one's walk terms in REGISTERS, and walks the rows twice from there:
//   count    one LDS add per (Gaussian, tile) instance;
//   reserve  one returning atomic per (workgroup, tile) on the tile's cursor: the workgroup's run inside the tile's bin;
//   emit     (depth bits << 32 | index) keys into the run, banded over the tile rows like k_tile_emit.
// The bins are the bin-by-tile path's: tile-major, fixed capacity (`bin_cap`, sized by the host from P / tiles with generous
// head-room), cursors cleared by the compositing kernel that consumes them -- no prefix sum over the tiles, no instance count
// on the host.  A tile that overflows its bin makes the compositing kernel report GSR_FAIL_OVERFLOW and the host falls back
// to the exact count -> scan -> emit path.  k_render_fwd<.., GSR_LIST_BINS_FULL> orders such a bin lazily, like a segment.
// ---------------------------------------------------------------------------------------------
#ifndef GSR_CURSOR64
#define GSR_CURSOR64 0             // 1: the tile cursor as a (slots, keys) pair behind one 64-bit atomic (for producers that pad their runs; the
                                   // compositing kernel copes with padding keys); 0: one 32-bit word, slots = keys -- measured 3 % faster on
                                   // S-1M-640's complete lists (4 290 against 4 170 it/s), 1-2 % on S-3M-cam
#endif
#define GSR_PBIN_THREADS 512
#define GSR_PBIN_KPT 4             // 2 048 Gaussians per workgroup: enough for the LDS counters to aggregate, two workgroups per CU
// Round 4 tried three other shapes of the reserve / emit half of this kernel, all measured on the MI355X and all slower or equal
// (HISTORY.md, round 4): (a) keys staged tile-major in 96 KB of LDS and flushed as whole 32-byte sectors, eight lanes per run -- one
// workgroup per CU is left, whose six barrier-separated phases have nobody to overlap with (same duration); (b) every (workgroup,
// tile) run padded to whole sectors with the key ~0 and ONE unbanded walk -- the walk is bound by the issue of its scattered 8-byte
// stores either way (48 k cycles against 42 k with two bands) and the padding stores cost another 40 k; (c) the reservation atomics
// issued early and consumed after the walk -- issuing them is what takes the time.  What stayed: four reservation atomics in flight
// per lane, workgroups staggered over the tiles, and a compositing kernel that copes with padding keys (GSR_CURSOR64).
__global__ void __launch_bounds__(GSR_PBIN_THREADS) k_preprocess_bin(PreArgs a, int bands)
{
    extern __shared__ uint32_t s_tb[];        // [0, ntiles) running count, [ntiles, 2 ntiles) where this workgroup's keys of the tile start
    __shared__ uint32_t s_pref[GSR_PBIN_THREADS];
    constexpr int KPT = GSR_PBIN_KPT, gpb = GSR_PBIN_KPT * GSR_PBIN_THREADS;
    const int nt = a.ntiles;
    uint32_t* s_cnt = s_tb;
    uint32_t* s_base = s_tb + nt;
    const int tid = threadIdx.x;
    GSR_T_DECL
    if (a.tile_order[0] != nullptr && blockIdx.x < 2) {      // native loop: this iteration's launch orders of the compositing kernels
        __shared__ uint32_t s_cls[GSR_BLOCK];
        tile_order_from_work(a.tile_work[blockIdx.x], a.tile_order[blockIdx.x], a.order_tiles, s_cls);
    }
    if (a.guard.poisoned()) return;
    for (int t = tid; t < nt; t += GSR_PBIN_THREADS) s_cnt[t] = 0u;
    if (blockIdx.x == 0 && tid == 0) {      // the null splat
        float4* nr = reinterpret_cast<float4*>(a.rec + (size_t)a.P * GSR_REC_STRIDE);
        nr[0] = make_float4(0.f, 0.f, 0.f, 0.f); nr[1] = nr[0]; nr[2] = nr[0];
    }
    WalkItem it[KPT];
#pragma unroll
    for (int k = 0; k < KPT; k++) {
        const int idx = blockIdx.x * gpb + k * GSR_PBIN_THREADS + tid;
        // (work lists: every 1024-Gaussian stretch counts as one block of surv_cap()'s accounting)
        const uint32_t vblock = (uint32_t)idx >> 10;
        WalkItem w = WalkItem{};          // (a local, copied into the register array: a pointer into it[] would put the array in scratch)
        preprocess_one<false>(a, idx, idx < a.P, nullptr, tid, vblock & (GSR_SURV_LISTS - 1), nullptr, &w);
        it[k] = w;
    }
    TileBinArgs ta = {};
    ta.gx = a.gx; ta.gy = a.gy;
    GSR_T_TICK(0)
    __syncthreads();
    GSR_T_TICK(1)
    walk_rows<KPT>(ta, it, 0, a.gy, s_pref, [&](int tile, unsigned long long) { atomicAdd(&s_cnt[tile], 1u); });
    GSR_T_TICK(2)
    __syncthreads();
    GSR_T_TICK(3)
    {
        // one returning atomic per (workgroup, tile), four in flight per lane, every workgroup starting at another tile; the cursor
        // is a (slots, keys) pair: both grow by the run's length here (a producer that pads its runs adds more slots than keys)
        const int rot = (int)((blockIdx.x * GSR_RESERVE_ROT) % (uint32_t)nt);
        unsigned long long* cur = reinterpret_cast<unsigned long long*>(a.tile_cursor);
        for (int t0 = tid; t0 < nt; t0 += 4 * GSR_PBIN_THREADS) {
            int tt[4];
            uint32_t c[4];
            unsigned long long old[4];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const int t = t0 + j * GSR_PBIN_THREADS;
                tt[j] = (t < nt) ? ((t + rot >= nt) ? t + rot - nt : t + rot) : -1;
                c[j] = (tt[j] >= 0) ? s_cnt[tt[j]] : 0u;
            }
#pragma unroll
            for (int j = 0; j < 4; j++) {
#if GSR_CURSOR64
                old[j] = (c[j] != 0u) ? atomicAdd(&cur[(size_t)tt[j] * (GSR_CURSOR_STRIDE / 2)], ((unsigned long long)c[j] << 32) | (unsigned long long)c[j]) : 0ull;
#else
                old[j] = (c[j] != 0u) ? (unsigned long long)atomicAdd(&a.tile_cursor[(size_t)tt[j] * GSR_CURSOR_STRIDE], c[j]) : 0ull;
#endif
            }
#pragma unroll
            for (int j = 0; j < 4; j++)
                if (tt[j] >= 0) { s_base[tt[j]] = (uint32_t)old[j]; s_cnt[tt[j]] = 0u; }
        }
    }
    GSR_T_TICK(4)
    const int bh = (a.gy + bands - 1) / bands;
    for (int b0 = 0; b0 < a.gy; b0 += bh) {
        __syncthreads();
        GSR_T_TICK(5)
        walk_rows<KPT>(ta, it, b0, min(a.gy, b0 + bh), s_pref, [&](int tile, unsigned long long key) {
            const uint32_t pos = s_base[tile] + atomicAdd(&s_cnt[tile], 1u);
            if (pos < (uint32_t)a.bin_cap) a.bins[(size_t)tile * (a.bin_cap + GSR_BIN_PAD) + pos] = key;
        });
        GSR_T_TICK(6)
    }
    GSR_T_FLUSH_W(32, GSR_PBIN_THREADS / 64)
}

// ---------------------------------------------------------------------------------------------
// K6  per-tile front-to-back compositing (replaces forward.cu:261-379 renderCUDA).
// One workgroup (4 waves) per 16x16 tile, one lane per pixel.  Batches of 256 splats are gathered
// once into LDS (44 B each: xy, conic, opacity, rgb, depth, id) and broadcast-read by every lane.
// ---------------------------------------------------------------------------------------------
// Which of the tile's four 8x8 pixel blocks (= waves) a staged splat can change: the exact x-extent of the ellipse
// q <= ln(255 o) (+ the same 0.02 slack as the tile culling) inside each of the tile's two bands of eight pixel rows --
// the span computation of row_span on an 8-row band -- against the two 8-pixel column ranges; widened by 0.01 px.
// (A bounding-box test leaves 13 % of a wave's list entries without a pixel that can use them; this costs two span
// evaluations per staged splat, once per tile, and shortens the walk of both compositing kernels.)
// Bit w set <=> wave w must look at the splat.  Not positive definite => all four.
__device__ __forceinline__ uint32_t quadrant_mask(float mx, float my, float A, float B, float C, float opacity, int X0, int Y0)
{
    const float det = A * C - B * B;
    if (!(A > 0.f && C > 0.f && det > 0.f)) return 0xFu;
#ifdef GSR_NO_CULL
    return 0xFu;
#endif
    const float qmax = (opacity > 0.f) ? (__logf(255.f * opacity) + 0.02f) : -1.f;
    if (qmax < 0.f) return 0u;
    const float twoq = 2.f * qmax, at = A * twoq, invA = __builtin_amdgcn_rcpf(A);
    const float dye = -B * __builtin_amdgcn_sqrtf(twoq * C * __builtin_amdgcn_rcpf(det)) * __builtin_amdgcn_rcpf(C);      // dy of the +x extreme point
    uint32_t m = 0;
#pragma unroll
    for (int band = 0; band < 2; band++) {
        const float dyh = my - (float)(Y0 + 8 * band), dyl = dyh - 7.f;           // d = mean - pixel over the band's rows
        const float dy1 = fminf(dyh, fmaxf(dyl, dye)), dy2 = fminf(dyh, fmaxf(dyl, -dye));
        const float disc1 = at - det * dy1 * dy1, disc2 = at - det * dy2 * dy2;
        if (fminf(disc1, disc2) < -1e-3f * at) continue;                             // the band lies outside the ellipse's y-extent
        const float dmax = (__builtin_amdgcn_sqrtf(fmaxf(disc1, 0.f)) - B * dy1) * invA;
        const float dmin = (-__builtin_amdgcn_sqrtf(fmaxf(disc2, 0.f)) - B * dy2) * invA;
        const float xl = mx - dmax - 0.01f - (float)X0, xh = mx - dmin + 0.01f - (float)X0;      // pixel interval relative to the tile
        if (xl <= 7.f && xh >= 0.f) m |= 1u << (2 * band);
        if (xl <= 15.f && xh >= 8.f) m |= 2u << (2 * band);
    }
    return m;
}

// The inner loop is shaped by one fact: a tile's walk is a long dependent chain and a wave issues at most one
// instruction every four cycles, VALU or scalar, so the kernel's duration is (list length) x (instructions per
// list entry) -- not bytes, not flops.
//   * the wave's list is consumed eight entries at a time: one 8-byte LDS read brings their indices into two
//     scalar registers, the bodies are unrolled, branch-free and their LDS reads independent of each other;
//     the last (fewer than eight) entries go through a plain tail loop;
//   * termination is folded into T: a finished pixel has T <= 0 (its true transmittance is -T), so
//     every later weight alpha*T vanishes by itself and no `done` flag has to be carried through the body;
//   * power > 0 (forward.cu:342) is folded into the `valid` predicate (a scalar AND, not a select on G);
//   * the conic is staged pre-multiplied, A2 = -a/2 log2e, B2 = -b log2e, C2 = -c/2 log2e, so that
//         power log2e = dx (A2 dx + B2 dy) + C2 dy dy
//     is two FMAs and three multiplies and feeds v_exp_f32 directly; K7 evaluates the identical expression, so
//     both passes see the same alpha bits;
//   * n_touched: eight popcounts are parked in eight lanes and leave as ONE atomic instruction per group.
// Tried and dropped (measured slower, single frame and with four frames in flight): two pixels per lane on the
// packed fp32 pipes with two waves per tile -- fewer VALU instructions per pixel, but half the waves to hide the
// chain's latency and twice the per-lane predicate bookkeeping (80 vs 60 us, 5.0 vs 5.2 k it/s at 4 frames).
// ---------------------------------------------------------------------------------------------
// Native loop: the tracking loss (descent_utils.py:85-123) and its pixel gradients are evaluated in the compositing
// kernel's epilogue, where the pixel's colour, depth and opacity are still in registers -- one launch and one pass over
// the images less per iteration.  Partial sums go to GSR_LOSS_SHARDS x {loss, dL/da, dL/db} accumulators (64 B apart),
// which the pose step adds up and clears.  out == nullptr: not fused (drop-in packages, gsr_tracking_loss).
// Complete lists (every forward without depth bounds: training, the first iteration of a refinement, the plain loop): all
// ~770 k visible Gaussians of S-1M-640 are binned, but the compositing kernel only ever stages the front of each tile's list
// (~380 k entries, 10 % of the instances).  Evaluating SH -> RGB for all of them beforehand read 148 MB of SH rows and cost
// 55 us per iteration (3 370 against 4 140 it/s without it), more than any other kernel of that path.  Instead the staging
// phase of k_render_fwd<.., GSR_LIST_EXACT> evaluates the colour of a splat the first time some tile stages it and leaves it
// in the splat's record (.w of the colour quad = 1: evaluated) for the other tiles and for the backward pass; `clamped` too.
// Two tiles staging the same splat at the same time both evaluate it and write the same values.  shs == nullptr: not lazy.
struct LazySH { const float* shs; const float* means; const float* campos; int D, M; uint8_t* clamped; float* rec; };

#define GSR_LOSS_SHARDS 16
struct FusedLoss {
    const float* gt_image; const float* gt_depth; const uint8_t* grad_mask; const float* exposure;
    float opacity_thr, depth_w; int monocular;
    float* dL_dimage; float* dL_ddepth; float* out;         // out: [GSR_LOSS_SHARDS][16] floats
    const float* conv;                                        // frozen after convergence, like k_tracking_loss
    int det;                                                  // deterministic option: the shard's first three 64-bit words, fixed point
};
__device__ __forceinline__ float sgnf(float d) { return (d > 0.f) ? 1.f : ((d < 0.f) ? -1.f : 0.f); }

// ---------------------------------------------------------------------------------------------
// Heavy tiles split across workgroups (round 5; native loop, speculative lists).
// A tile is one workgroup and a pixel's compositing is a dependent chain: on a structured scene (a dense object, a wall seen at a
// grazing angle) a handful of tiles need lists ten times the mean, ONE of their four waves walks them while the other three wait
// at the batch barriers, and both compositing kernels last as long as that wave (S-room-640: K6 576 us, K7 676 us for work that
// would take ~100 us spread evenly; phase clocks in profiles/r05_phase_clocks.md).  Such a tile is cut into `nseg` DEPTH RANGES,
// one workgroup ("segment") each:
//   * every segment derives the same nseg - 1 depth pivots from the same 1 024-key sample of the tile's bin (same arithmetic on
//     the same data: no communication), gathers the keys of its own range, orders them (<= 2 048) and stages their records;
//   * pass A walks them for the per-pixel product Tl of (1 - alpha) over the valid entries only -- no colours, no termination --
//     and publishes it; a segment then multiplies its predecessors' products in segment order into Ts, its pixels' transmittance
//     at its first entry; pass C is the normal walk started at Ts.  Transmittance is carried as Ts x Tl (Tl restarts at 1 in every
//     segment) and a pixel terminates where Ts x Tl x (1 - alpha) < 1e-4: by monotonicity that is the case somewhere in segment s
//     exactly if Ts(s + 1) < 1e-4, so every later segment knows a pixel is finished from the products alone;
//   * a segment leaves a record per pixel (Ts, signed end transmittance, its colour / depth sums, last contributor, depth
//     needed) and its ordered index list at its place in the tile's list; the segment that finishes LAST (a ticket per tile)
//     adds the records up in segment order and runs the normal epilogue (images, fused loss, depth bounds, verification);
//   * k_render_bwd_mfma walks the segments in parallel too: segment s starts behind its last entry with T = Ts(s + 1) and the
//     "composited behind me" value (sum of the later segments' colour sums . dL/dpixel) / Ts(s + 1).
// Against the unsplit walk the results differ by rounding only (T as a product of per-segment products instead of one running
// product): the deterministic option therefore never splits, and parity against the CPU restatement of the reference is tested with splitting live
// (tests/test_gpu_split.py).  A block of the launch is (tile, segment, nseg) from `list`; which tiles are split how far is decided
// on the device from the work the previous iteration's forward measured (seg_list_build).
// Waiting is only ever for LOWER-numbered blocks of the same launch (a tile's segments sit in consecutive blocks, ascending), which
// the dispatcher has started earlier: no deadlock as long as workgroups are started in block order; every wait is bounded anyway.
// ---------------------------------------------------------------------------------------------
#define GSR_SEG_REC_Q 10           // floats per pixel and segment: Tl, Ts, end T (signed), r, g, b, depth sums, last contributor, depth needed, work
#define GSR_SEG_SHARE_MAX 1365     // a tile is only split while (its keys / nseg) stays below this: a range must fit the in-LDS sort (2 048) with room for sampling noise
struct SegCtl {
    const uint32_t* list;          // per block: tile | segment << 16 | nseg << 24; ~0: nothing to do.  nullptr: no splitting, blockIdx -> tile as before
    uint32_t* cnt;                 // per block: (epoch << 16) | keys of the segment + 1 (low half 0: its tile was not split after all)
    uint32_t* pub;                 // per block: (epoch << 2) | 1 once the segment's Tl are out
    float* rec;                    // per block: GSR_SEG_REC_Q x 256 floats
    uint32_t* ticket;              // per tile: [2 t] segments that have read the bin's cursor, [2 t + 1] segments that have finished
    uint32_t* nosplit;             // per tile: forwards this tile still goes unsplit (a range once exceeded the in-LDS sort)
    uint32_t epoch;                // tag of this launch's group (flags of earlier launches never match)
    uint32_t* len;                 // per tile, out (nullable): list entries this forward ordered for the tile -- how long its next bin will be, roughly
    uint32_t hold_after;           // (rides along: after how many failed verifications in a call a tile keeps its complete list for a while -- see tile_hold)
    // (rides along too) widened bounds, see dilate_bounds: zb_own_used = the bounds this forward's tiles recorded THEMSELVES last time (before
    // any widening), nodilate = per tile, forwards it still goes without widening.  A tile whose bin overflows under a bound it took from
    // a neighbour falls back to its own bound and is retried on the device like a failed verification, instead of failing the forward.
    const float* zb_own_used; uint32_t* nodilate;
};
// The NEXT iteration's launch list is built by one extra workgroup of k_render_bwd_mfma (block `block`, which does nothing else) from the
// work this iteration's forward measured -- next to the longest kernel of the loop, off everybody's critical path (in the preprocess
// kernel, whose workgroups are all resident from the start, it ran last and cost the loop 3.4 us).  Two lists: a launch walks one while
// it builds the other.  list == nullptr: nothing to build.
struct SegBuild {
    const uint32_t* work; uint32_t* order; uint32_t* list; uint32_t* nosplit; int ntiles, budget, block; const uint32_t* len;
    // The same workgroup also widens the depth bounds this group's forward recorded where they jump (zb nullable): a tile next to one
    // that needed to look much deeper -- or did not saturate at all -- takes its neighbour's bound.  An object's silhouette in front of a
    // wall two metres behind moves by a fraction of a pixel per iteration; the tile it moves INTO had saturated on the object and now
    // has a pixel that needs the wall: a failed verification, i.e. a wasted forward, almost every iteration (S-room-640: 28 of 50).
    // Deeper bounds only make lists longer: results cannot depend on it.
    float* zb; float* zbc; int gx, gy, sbx;
    float* zb_own; uint32_t* nodilate;      // out: every tile's own bound (before widening); per tile: forwards it still goes without widening
    int split_ok;                           // 0: this group's work figures are not a speculative forward's -- the list it builds splits nobody
    uint32_t* host_total;                   // out (nullable, pinned host memory): blocks the list holds -- the host sizes later launches by it
};
#ifndef GSR_BOUND_DILATE_RATIO
#define GSR_BOUND_DILATE_RATIO 1.25f
#endif
#define GSR_DILATE_INF_MAX_LEN 2048u
#ifndef GSR_DILATE_MAX_LEN
#define GSR_DILATE_MAX_LEN 6144u
#endif
__device__ __forceinline__ void dilate_bounds(const SegBuild& sb, float* scratch /* ntiles floats */)
{
    const int nt = sb.gx * sb.gy;
    for (int t = threadIdx.x; t < nt; t += blockDim.x) {
        const int tx = t % sb.gx, ty = t / sb.gx;
        const float mine = sb.zb[t];
        float nb = 0.f;
        for (int dy = -1; dy <= 1; dy++)
            for (int dx = -1; dx <= 1; dx++) {
                const int x = tx + dx, y = ty + dy;
                if ((dx != 0 || dy != 0) && x >= 0 && x < sb.gx && y >= 0 && y < sb.gy) {
                    const float z = sb.zb[y * sb.gx + x];
                    // (a neighbour WITHOUT a bound -- it did not saturate -- hands that on only if its own complete list, which it has just
                    // walked to the end, is short: "no bound" means the complete list, and next to a dense object that is a hundred times
                    // the needed one and overflows the bin -- S-1M-640-object: bins of 8 192 against complete lists of 100 000)
                    if (z < __builtin_huge_valf() || sb.len[y * sb.gx + x] <= GSR_DILATE_INF_MAX_LEN) nb = fmaxf(nb, z);
                }
            }
        // (... and only where the longer list is affordable: this tile's list grows roughly in proportion to the depth it covers; a tile on a
        // dense object that took the bound of its neighbour in the sparse background behind would bin the whole object -- an overflowing bin)
        const float mylen = (float)sb.len[t];
#ifndef GSR_DILATE_INF_OWN_MAX
#define GSR_DILATE_INF_OWN_MAX 0xFFFFFFFFu      // (experiment, round 6: a BOUNDED tile takes "no bound" from a neighbour only if its own needed list is at most this long)
#endif
        const bool affordable = (nb < __builtin_huge_valf()) ? (mine > 0.f && mylen * (nb / mine) <= (float)GSR_DILATE_MAX_LEN)
                                                              : (!(mine < __builtin_huge_valf()) || sb.len[t] <= GSR_DILATE_INF_OWN_MAX);
        uint32_t hold = sb.nodilate[t];      // (a tile whose widened bin overflowed goes without for a while: k_render_fwd set this)
        if (hold != 0u) sb.nodilate[t] = hold - 1u;
        sb.zb_own[t] = mine;
        scratch[t] = (nb > mine * GSR_BOUND_DILATE_RATIO + 0.25f && affordable && hold == 0u) ? nb : mine;
    }
    __syncthreads();
    for (int t = threadIdx.x; t < nt; t += blockDim.x) {
        const float v = scratch[t];
        if (v != sb.zb[t]) {
            sb.zb[t] = v;
            const int tx = t % sb.gx, ty = t / sb.gx;
            atomicMax(reinterpret_cast<int*>(sb.zbc) + (ty >> 2) * sb.sbx + (tx >> 2), __float_as_int(v));
        }
    }
}
__device__ __forceinline__ void seg_store(float* p, float v) { __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
__device__ __forceinline__ float seg_load(const float* p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
__device__ __forceinline__ void seg_store_u(uint32_t* p, uint32_t v) { __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
__device__ __forceinline__ uint32_t seg_load_u(const uint32_t* p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }

// Record layout: what the walk reads per list entry is a (16 B), the first half of b (8 B) and c (16 B), and the fields sit
// next to each other as operand PAIRS: (x, y) - (px, py), (B2, C2) * dy, (r, g) * w, (b, depth) * w.  (The build switches the packed fp32 instructions
// off: two plain operations each, the same bits; pose loop +0.7 % on S-1M-640, -0.9 % on S-3M-cam.)
typedef float gsr_f32x2 __attribute__((ext_vector_type(2)));
typedef float gsr_f32x4 __attribute__((ext_vector_type(4)));
struct SplatLDS {
    float4 a[GSR_BLOCK];   // x, y, B2, C2
    float4 b[GSR_BLOCK];   // A2, opacity | id (bits), quadrant mask (bits)
    float4 c[GSR_BLOCK];   // r, g, b, depth
    alignas(8) uint8_t list[4][GSR_BLOCK];   // per wave: staged splats that can touch its 8x8 block, in list order
};

// Where the tile's list comes from:
//   GSR_LIST_SORTED  point_list[ranges[tile]] is already in (depth, index) order (re-compositing a forward's lists);
//   GSR_LIST_BINS    fixed-capacity bin of the native loop's speculative iterations (<= GSR_LSORT_CAP keys, appended by
//                    k_preprocess): sorted here in LDS in one go;
//   GSR_LIST_EXACT   the tile's segment of the exact bins (k_tile_emit), any length: ordered lazily, slice by slice.
#define GSR_LIST_SORTED 0
#define GSR_LIST_BINS 1
#define GSR_LIST_EXACT 2
#define GSR_LIST_BINS_FULL 3       // a bin like GSR_LIST_BINS holding the tile's COMPLETE list (k_preprocess_bin): treated like a segment
                                   // of the exact bins -- lazy slices above one register sort's worth of keys (256), lazy SH colours
#define GSR_SEL_BITS 11            // radix of the selection histogram (2048 counters, aliased onto the key buffer)
#ifndef GSR_SLICE_WANT0
#define GSR_SLICE_WANT0 200        // sample_slice: keys the first slice aims at (<= 256 sort in registers), the second, the later ones
#endif
#define GSR_SLICE_WANT1 448
#define GSR_SLICE_WANT2 1800

// Bitonic sort of s_keys[0, npow) (npow a power of two >= 64), ascending; all GSR_BLOCK threads.
// (measured: a rank sort and a variant with wave-local steps and 3 barriers instead of 45 are no faster --
// with five workgroups per CU sorting at the same time the step is bound by its ~25 VALU instructions)
__device__ __forceinline__ void lds_bitonic_sort(unsigned long long* s_keys, int npow)
{
    const int tid = threadIdx.x;
    for (int k = 2; k <= npow; k <<= 1)
        for (int j = k >> 1; j > 0; j >>= 1) {
            for (int q = tid; q < (npow >> 1); q += GSR_BLOCK) {      // one compare-exchange per lane
                const int i = ((q & ~(j - 1)) << 1) | (q & (j - 1)), l = i | j;
                const unsigned long long a0 = s_keys[i], a1 = s_keys[l];
                const bool up = (i & k) == 0;
                if ((a0 > a1) == up) { s_keys[i] = a1; s_keys[l] = a0; }
            }
            __syncthreads();
        }
}

// At most GSR_BLOCK keys (one per thread, ~0 = none; real keys are unique): every wave sorts its 64 keys in REGISTERS (bitonic
// network over the lanes: 21 compare-exchange steps through ds_bpermute, no barrier, no LDS traffic of its own), the four
// sorted runs meet in s_keys, and every thread finds its key's final place by counting, in each of the other three runs,
// the keys below its own (6-step binary searches).  Three barriers instead of the 36 of the LDS network on 256 keys: ~5 k
// instead of ~16 k cycles per wave on the native loop's bins (a fifth of k_render_fwd's time).  s_keys[0, total) sorted on return.
__device__ __forceinline__ void sort_block_keys(unsigned long long key, unsigned long long* s_keys)
{
    const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
#pragma unroll
    for (int k = 2; k <= 64; k <<= 1)
#pragma unroll
        for (int j = k >> 1; j > 0; j >>= 1) {
            const unsigned long long other = __shfl_xor(key, j, 64);
            const bool take_min = ((lane & j) == 0) == ((lane & k) == 0);      // lower lane of an ascending pair, or upper lane of a descending one
            key = (take_min == (other < key)) ? other : key;
        }
    s_keys[tid] = key;
    __syncthreads();
    int rank = lane;
#pragma unroll
    for (int w = 0; w < 4; w++) {
        if (w == wv) continue;
        const unsigned long long* run = s_keys + w * 64;
        int pos = 0;
#pragma unroll
        for (int step = 32; step > 0; step >>= 1)
            if (run[pos + step - 1] < key) pos += step;
        rank += pos + ((pos == 63 && run[63] < key) ? 1 : 0);
    }
    __syncthreads();
    if (key != ~0ull) s_keys[rank] = key;
    __syncthreads();
}

// GSR_LIST_EXACT: picks the next slice of a tile's unordered segment keys[0, total).  Keys are unique (the index is part
// of them).  Among the keys above `lo` (all of them when `first`) finds a threshold `hi` such that the number m of keys in
// (lo, hi] satisfies 1 <= m <= limit and, unless the keys run out of distinguishing bits earlier, m >= limit / 4:
// most-significant-digit radix selection, GSR_SEL_BITS bits per pass over the segment (two or three passes for depths a
// few octaves apart).  Block-uniform result; s_hist: 2^GSR_SEL_BITS counters; all threads must call.
__device__ __forceinline__ void select_slice(const unsigned long long* __restrict__ keys, int total, bool first, unsigned long long lo,
                                             int limit, uint32_t* s_hist, unsigned long long& hi, int& m)
{
    __shared__ uint32_t s_part[4];
    __shared__ int s_best[2];            // largest digit that still fits, and the count accepted through it
    const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
    const int minimum = limit >> 2;
    unsigned long long prefix = 0ull;
    int prefix_bits = 0, accepted = 0;
    for (;;) {
        const int dbits = min(GSR_SEL_BITS, 64 - prefix_bits), shift = 64 - prefix_bits - dbits;
        const int nbins = 1 << dbits;
        for (int i = tid; i < (1 << GSR_SEL_BITS); i += GSR_BLOCK) s_hist[i] = 0u;
        if (tid == 0) { s_best[0] = -1; s_best[1] = accepted; }
        __syncthreads();
        for (int i = tid; i < total; i += GSR_BLOCK) {
            const unsigned long long k = keys[i];
            const bool in = (first || k > lo) && k != ~0ull && (prefix_bits == 0 || (k >> (64 - prefix_bits)) == prefix);      // (~0: padding)
            if (in) atomicAdd(&s_hist[(uint32_t)(k >> shift) & (uint32_t)(nbins - 1)], 1u);
        }
        __syncthreads();
        // thread t owns bins [8 t, 8 t + 8): exclusive prefix of the per-thread sums, then a local walk
        uint32_t c[8], mine = 0u;
#pragma unroll
        for (int q = 0; q < 8; q++) { c[q] = s_hist[8 * tid + q]; mine += c[q]; }
        uint32_t incl = mine;
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
            const uint32_t o = __shfl_up(incl, off, 64);
            if (lane >= off) incl += o;
        }
        if (lane == 63) s_part[wv] = incl;
        __syncthreads();
        uint32_t run = (uint32_t)accepted + incl - mine;
        for (int w = 0; w < wv; w++) run += s_part[w];
        int best = -1, best_cnt = 0;
#pragma unroll
        for (int q = 0; q < 8; q++) {
            run += c[q];
            if (8 * tid + q < nbins && run <= (uint32_t)limit) { best = 8 * tid + q; best_cnt = (int)run; }
        }
        // cumulative counts are monotone, so the qualifying digits form a prefix: the largest one wins
        if (best >= 0) atomicMax(&s_best[0], best);
        __syncthreads();
        if (best >= 0 && best == s_best[0]) s_best[1] = best_cnt;
        __syncthreads();
        const int d = s_best[0], acc = s_best[1];
        __syncthreads();
        if (acc >= minimum || shift == 0) {
            // everything below the current prefix's digit d + 1
            const unsigned long long top = ((prefix << dbits) + (unsigned long long)(d + 1)) << shift;      // first key NOT taken
            hi = top - 1ull;
            m = acc;
            return;
        }
        accepted = acc;
        prefix = (prefix << dbits) | (unsigned long long)(d + 1);
        prefix_bits += dbits;
    }
}

// Lazy slices, round 4: pick the next slice with ONE pass over the tile's keys instead of two to four.
// select_slice above finds an exact rank threshold by most-significant-digit radix selection: every pass re-reads the tile's ~2 800
// keys from global memory and pushes each through an LDS atomic (64 k of a wave's 154 k cycles on S-1M-640's complete lists, 141 k of
// 237 k on S-3M-cam's; 157 MB of HBM traffic per launch for 27 MB of keys).  But a slice does not need an exact rank -- any depth
// threshold that admits "a couple of hundred" keys will do.  So: 1 024 keys of the segment (sixteen runs of 64 spread over it: a sample
// that is unrelated to depth) go through LDS into registers, sixteen per lane, in EVERY wave; each wave bisects on the depth bits
// until the sample count below the threshold matches the wanted share (wave ballots + scalar popcounts: no barrier, no atomics,
// the four waves arrive at the same threshold because they run the same arithmetic on the same data); then one coalesced pass over
// all keys gathers those at or below the threshold into s_keys with a ballot prefix per wave (one LDS atomic per wave and 256 keys).
// Returns the number gathered (block-uniform; 0 = sample empty, > cap = the caller must retry with a smaller share or fall back to
// select_slice -- thousands of keys sharing one depth).  hi = the slice's upper key bound.  s_samp: 1 024 words of LDS.
__device__ __forceinline__ int sample_slice(const unsigned long long* __restrict__ keys, int total /* slots, padding keys ~0 included */, bool first, unsigned long long lo, int remaining,
                                            int want, int cap, uint32_t* s_samp, unsigned long long* s_keys, unsigned long long& hi GSR_T_PARAMS)
{
    __shared__ uint32_t s_fill;
    const int tid = threadIdx.x, lane = tid & 63;
    // (sixteen runs of 64 keys spread evenly over the segment, not its first 1 024 keys: arrival order is only unrelated to depth while
    // the MAP's order is unrelated to space -- on a Morton-sorted map every workgroup's run in a tile holds one depth range, the head of
    // the segment says little about the rest, and the kernel took 94 instead of 75 us on S-1M-640, 212 instead of 114 on S-3M-cam)
#ifndef GSR_SAMPLE_RUN
#define GSR_SAMPLE_RUN 64          // keys per run of the sample (a power of two, 64 ... 1 024 = the head of the segment; measured on S-3M-cam's
                                   // complete lists, random / Morton order: 64 -> 127 / 130 us, 256 -> 126 / 131, 1 024 -> 120 / 218)
#endif
    const int nruns = (total + GSR_SAMPLE_RUN - 1) / GSR_SAMPLE_RUN;
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const int i = tid + GSR_BLOCK * j;
        const int run = i / GSR_SAMPLE_RUN;
        const int pos = ((nruns <= 1024 / GSR_SAMPLE_RUN) ? run : (int)(((long long)run * nruns) / (1024 / GSR_SAMPLE_RUN))) * GSR_SAMPLE_RUN + (i & (GSR_SAMPLE_RUN - 1));
        uint32_t d = 0xFFFFFFFFu;
        if (pos < total) {
            const unsigned long long k = keys[pos];
            if (first || k > lo) d = (uint32_t)(k >> 32);
        }
        s_samp[i] = d;
    }
    if (tid == 0) s_fill = 0u;
    __syncthreads();
    uint32_t v[16];
#pragma unroll
    for (int q = 0; q < 4; q++) {
        const uint4 x = reinterpret_cast<const uint4*>(s_samp)[lane + 64 * q];
        v[4 * q] = x.x; v[4 * q + 1] = x.y; v[4 * q + 2] = x.z; v[4 * q + 3] = x.w;
    }
    int nvalid = 0;
    uint32_t vmin = 0xFFFFFFFFu, vmax = 0u;
#pragma unroll
    for (int q = 0; q < 16; q++) {
        const bool ok = v[q] != 0xFFFFFFFFu;
        nvalid += (int)__popcll(__ballot(ok));
        vmin = min(vmin, v[q]);
        vmax = ok ? max(vmax, v[q]) : vmax;
    }
    if (nvalid == 0) { hi = lo; return 0; }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) {
        vmin = min(vmin, (uint32_t)__shfl_xor((int)vmin, off, 64));
        vmax = max(vmax, (uint32_t)__shfl_xor((int)vmax, off, 64));
    }
    uint32_t pivot;
    if (remaining <= want) pivot = 0xFFFFFFFEu;              // everything that is left
    else {
        // share of the sample that stands for `want` of the `remaining` keys; accepted up to an eighth above it
        const int r = max(1, min(nvalid, (int)(((long long)want * nvalid + remaining - 1) / remaining)));
        const int tol = r >> 3;
        uint32_t lo_b = (uint32_t)__builtin_amdgcn_readfirstlane((int)vmin), hi_b = (uint32_t)__builtin_amdgcn_readfirstlane((int)vmax);
        // Bisection on the depth bits: invariant count(<= hi_b) >= r, count(< lo_b) < r; it stops as soon as a probe's count lies in
        // [r, r + r / 8] -- eight to ten probes, each sixteen compares per lane and their ballots' popcounts on the scalar unit.
        // (Interpolating the probe between the bracket's counts, on the depth values, needs three or four probes and measured the
        // same: the phase is the sample's round trip through memory, not the probes.)
        while (lo_b < hi_b) {
            const uint32_t mid = lo_b + ((hi_b - lo_b) >> 1);
            int c = 0;
#pragma unroll
            for (int q = 0; q < 16; q++) c += (int)__popcll(__ballot(v[q] <= mid));
            if (c >= r) { hi_b = mid; if (c <= r + tol) break; }
            else lo_b = mid + 1u;
        }
        pivot = hi_b;
    }
    hi = ((unsigned long long)pivot << 32) | 0xFFFFFFFFull;
    GSR_T_TICK_O(4)
    for (int i0 = 0; i0 < total; i0 += 4 * GSR_BLOCK) {
        unsigned long long k[4];
        bool in[4];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int i = i0 + j * GSR_BLOCK + tid;
            k[j] = (i < total) ? keys[i] : 0ull;
            in[j] = i < total && (first || k[j] > lo) && (uint32_t)(k[j] >> 32) <= pivot;
        }
        // one LDS atomic per wave and 1 024 keys: the four ballots' counts are reserved together
        unsigned long long mk[4];
        uint32_t cnt4 = 0u;
#pragma unroll
        for (int j = 0; j < 4; j++) { mk[j] = __ballot(in[j]); cnt4 += (uint32_t)__popcll(mk[j]); }
        if (cnt4 != 0u) {                                    // wave-uniform
            uint32_t base = 0u;
            if (lane == 0) base = atomicAdd(&s_fill, cnt4);
            base = (uint32_t)__builtin_amdgcn_readfirstlane((int)base);
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const uint32_t pos = base + (uint32_t)__popcll(mk[j] & ((1ull << lane) - 1ull));
                if (in[j] && pos < (uint32_t)cap) s_keys[pos] = k[j];
                base += (uint32_t)__popcll(mk[j]);
            }
        }
    }
    __syncthreads();
    GSR_T_TICK_O(6)
    return (int)s_fill;
}

// (5 workgroups per CU keep every tile of a 640x480 image resident in one round: 96 registers.  The slice-ordering variant
// with the n_touched counters needs a few more and gets 4 per CU rather than spilling.)
template <bool TOUCHED, int LIST>
__global__ void __launch_bounds__(GSR_BLOCK, (TOUCHED && LIST != GSR_LIST_SORTED) ? 4 : 5) k_render_fwd(uint2* __restrict__ ranges,
                                                          uint32_t* __restrict__ point_list,
                                                          const unsigned long long* __restrict__ bins,
                                                          uint32_t* __restrict__ tile_cursor,
                                                          int W, int H, int gx,
                                                          int ntiles, const float* rec, const float* __restrict__ bg,
                                                          float* __restrict__ out_color, float* __restrict__ out_depth,
                                                          float* __restrict__ out_alpha, uint32_t* __restrict__ n_contrib,
                                                          int* __restrict__ n_touched, float* __restrict__ zb_next,
                                                          const float* __restrict__ zb_used, uint32_t* __restrict__ fail,
                                                          float margin_mul, float margin_add, float* __restrict__ zbc_next,
                                                          int sbx, FusedLoss fl, const uint32_t* __restrict__ tile_order,
                                                          uint32_t* __restrict__ tile_work, int bin_cap, LazySH lz, uint32_t fail_tag,
                                                          uint32_t* __restrict__ tile_total, int pack_qm, uint32_t* __restrict__ tile_hold, SegCtl sg)
{
    // (tile_hold, nullable, native loop: per tile, for how many more forwards it goes without a depth bound after it failed a
    // verification -- see where the bounds are recorded)
    // (pack_qm: the sorted index list carries every staged splat's quadrant mask for this tile in bits 28-31 of its entry -- written
    // below, read by k_render_bwd_mfma's staging, which then needs neither the splat's record nor the span arithmetic again.
    // The host sets it when P < 2^28.)
    // (tile_total, nullable, ntiles words: GSR_LIST_BINS_FULL leaves every tile's complete instance count there; their sum is the
    // forward's num_rendered)
    // (fail: the word a failed verification is reported in -- the loop's poison word with fail_tag = this group's tag << 2, see
    // LoopGuard; the drop-in speculation's flag word with fail_tag = 0)
    // (tile_cursor: GSR_LIST_BINS the per-tile append cursors; GSR_LIST_EXACT the tile_offset array of k_tile_scan)
    __shared__ SplatLDS s;
    __shared__ float s_zmax[4];
    __shared__ unsigned long long s_keys[LIST != GSR_LIST_SORTED ? GSR_LSORT_CAP : 1];
    GSR_T_DECL
    // (tile_order: the native loop's work-balanced launch order, see tile_order_from_work; otherwise XCD-contiguous runs of tiles)
    // (sg.list: this launch's blocks are (tile, segment) pairs, heaviest tiles first -- see SegCtl; nseg == 1: an ordinary tile)
    int tile;
    uint32_t seg = 0u, nseg = 1u;
    if (LIST == GSR_LIST_BINS && sg.list != nullptr) {
        const uint32_t e = sg.list[blockIdx.x];
        if (e == 0xFFFFFFFFu) return;
        tile = (int)(e & 0xFFFFu); seg = (e >> 16) & 0xFFu; nseg = e >> 24;
    } else tile = tile_order ? (int)tile_order[blockIdx.x] : xcd_remap(blockIdx.x, ntiles);
    const int tx = tile % gx, ty = tile / gx;
    const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
    const int px = tx * GSR_TILE + (wv & 1) * 8 + (tid & 7), py = ty * GSR_TILE + (wv >> 1) * 8 + ((tid >> 3) & 7);
    const bool inside = px < W && py < H;
    const int pix_id = W * py + px;
    const float pxf = (float)px, pyf = (float)py;
    uint2 range;
    int nslots = 0;      // memory extent of the tile's unordered keys (>= their number: padding keys ~0 in fixed-capacity complete bins)
    constexpr bool kBins = (LIST == GSR_LIST_BINS || LIST == GSR_LIST_BINS_FULL);
    constexpr bool kFull = (LIST == GSR_LIST_EXACT || LIST == GSR_LIST_BINS_FULL);      // complete lists: lazy ordering, lazy SH colours
    if (kBins) {
        // one lane reads the tile's cursor and clears it for the next iteration's appends (no memset); everybody else
        // gets the count through LDS
        // (word 0: slots handed out in the bin; word 1, GSR_LIST_BINS_FULL only: the keys among them -- k_preprocess_bin pads every
        // workgroup's run to whole 32-byte sectors with the key ~0)
        __shared__ uint32_t s_cursor[2];
        // (requesting the bin's first 256 keys here, next to the cursor, instead of one round trip behind it: measured, no difference)
        if (tid == 0) {
            const uint32_t slots = tile_cursor[tile * GSR_CURSOR_STRIDE];
            s_cursor[0] = slots;
            s_cursor[1] = (LIST == GSR_LIST_BINS_FULL && GSR_CURSOR64) ? tile_cursor[tile * GSR_CURSOR_STRIDE + 1] : slots;
            bool clear = true;
            if (LIST == GSR_LIST_BINS && nseg > 1u) {          // a split tile: every segment reads the cursor, the last reader clears it
                asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
                clear = atomicAdd(&sg.ticket[2 * tile], 1u) == nseg - 1u;
                if (clear) sg.ticket[2 * tile] = 0u;
            }
            if (clear) {
                tile_cursor[tile * GSR_CURSOR_STRIDE] = 0u;
                if (LIST == GSR_LIST_BINS_FULL) tile_cursor[tile * GSR_CURSOR_STRIDE + 1] = 0u;
            }
        }
        __syncthreads();
        range.x = (uint32_t)tile * (uint32_t)(bin_cap + GSR_BIN_PAD);
        range.y = range.x + s_cursor[1];
        nslots = (int)s_cursor[0];
    } else if (LIST == GSR_LIST_EXACT) {
        range.x = tile_cursor[tile];
        range.y = tile_cursor[tile + 1];
    } else range = ranges[tile];
    // RECOUNT (TOUCHED on GSR_LIST_SORTED: gsr_refine's closing n_touched pass over the lists of a forward that has already produced
    // the images): the walk follows the forward's own per-pixel decisions -- pixel p looks at list positions 1 .. n_contrib[p], with
    // the same blend tests and no termination test of its own -- and writes nothing but the counters.  The forward may have been a
    // SPLIT one (transmittance carried as a product of per-range products: another rounding, so this pass's own termination could
    // differ by a splat; and a range that found every pixel finished never wrote its part of the list, so positions beyond the
    // tile's deepest contributor may hold stale indices): nothing beyond that position is read.
    constexpr bool RECOUNT = TOUCHED && LIST == GSR_LIST_SORTED;
    uint32_t rc_lim = 0u;
    if (RECOUNT) {
        __shared__ uint32_t s_rc[4];
        rc_lim = inside ? n_contrib[pix_id] : 0u;
        uint32_t mx = rc_lim;
#pragma unroll
        for (int off = 32; off > 0; off >>= 1) mx = max(mx, (uint32_t)__shfl_xor((int)mx, off, 64));
        if (lane == 0) s_rc[wv] = mx;
        __syncthreads();
        range.y = min(range.y, range.x + max(max(s_rc[0], s_rc[1]), max(s_rc[2], s_rc[3])));
    }
    const int total = (int)(range.y - range.x);
    if (!kBins) nslots = total;
#ifdef GSR_DBG_TILE
    if (LIST == GSR_LIST_BINS && fail_tag != 0u && tid == 0 && tile == GSR_DBG_TILE) { fail[4] = (uint32_t)nslots; fail[5] = __float_as_uint(zb_used ? zb_used[tile] : -1.f); fail[6] = sg.hold_after; fail[7] = tile_hold ? tile_hold[tile] : 0xFFFFu; }
#endif
    // (one plain store per tile.  A grand total added up here with one atomic per tile cost 16 us: 1 200 same-address atomics queue
    // up at the memory side and every workgroup's next barrier waits for its own)
    if (LIST == GSR_LIST_BINS_FULL && tile_total != nullptr && tid == 0) tile_total[tile] = (uint32_t)total;
    int walked = 0, overhead = 0;      // -> tile_work: groups of eight this wave composited; staging / ordering cost in the same unit

    // A tile the launch list wants split (SegCtl) is only split if its bin allows it -- no overflow, more than one staging batch, and
    // a share per segment that fits the in-LDS sort.  Every segment takes this decision from the same numbers; if it is "no",
    // segment 0 handles the tile like any other and says so in its count word (k_render_bwd_mfma reads it), the others leave.
    bool split = false;
    if (LIST == GSR_LIST_BINS && nseg > 1u) {
        split = nslots <= bin_cap && total > GSR_BLOCK && total <= (int)nseg * GSR_SEG_SHARE_MAX;
        if (!split) {
            if (seg != 0u) return;
            nseg = 1u;
            if (tid == 0) seg_store_u(&sg.cnt[blockIdx.x], sg.epoch << 16);
        }
    }

    // A bin longer than the in-LDS sort takes (a tile that does not saturate -- the edge of the scene's coverage, a
    // semi-transparent region -- has no depth bound and gets its complete list) is ordered lazily, slice by slice, like a
    // segment of the exact bins; only a bin that overflowed its capacity fails the forward.
    const bool lazy = !split && ((LIST == GSR_LIST_EXACT) || (LIST == GSR_LIST_BINS && total > GSR_LSORT_CAP) || (LIST == GSR_LIST_BINS_FULL && nslots > GSR_BLOCK));
    if (kBins && nslots > bin_cap) {          // block-uniform: entries were dropped; the host redoes the forward with complete lists
        if (tid == 0 && LIST == GSR_LIST_BINS && sg.zb_own_used != nullptr && zb_used != nullptr && zb_next != nullptr && sg.zb_own_used[tile] < zb_used[tile]) {
            // the bound this tile was binned with was a neighbour's (dilate_bounds): back to its own, which held a list that fitted, no widening
            // for a while, and the forward fails like a verification -- the group behind this one retries it on the device
            const float own = sg.zb_own_used[tile];
#ifndef GSR_NODILATE_HOLD
#define GSR_NODILATE_HOLD 64u
#endif
            sg.nodilate[tile] = GSR_NODILATE_HOLD;
            zb_next[tile] = own;
            atomicMax(reinterpret_cast<int*>(zbc_next) + (ty >> 2) * sbx + (tx >> 2), __float_as_int(own));
            atomicMax(fail, fail_tag | GSR_FAIL_BOUND);
        } else
        if (tid == 0) {
            atomicMax(fail, fail_tag | GSR_FAIL_OVERFLOW);
            if (fail_tag != 0u) { fail[2] = (uint32_t)tile; fail[3] = (uint32_t)nslots; }      // (native loop, diagnostics: pose-state words 42 / 43, free otherwise -- GSR_REFINE_LOG_REDO prints them)
            // The group enqueued behind this one bins with the bounds THIS forward records (it is the device-side retry): a tile
            // that leaves without recording one would hand it whatever the buffer held before -- a stale per-tile bound next to
            // superblock maxima this tile never contributed to, i.e. lists that are no longer depth-prefixes, from which a pixel can
            // saturate on the wrong entries without failing its verification (found by the bit-for-bit fuzz of the deterministic
            // option, round 3: poses 1e-4 off on scenes of 0.2 m splats).  No bound: the retry gets this tile's complete list (and,
            // if that overflows its bin as well, fails in turn: the host then bins exactly).
            if (zb_next != nullptr) {
                zb_next[tile] = __builtin_huge_valf();
                atomicMax(reinterpret_cast<int*>(zbc_next) + (ty >> 2) * sbx + (tx >> 2), __float_as_int(__builtin_huge_valf()));
            }
        }
        return;
    }
    if (kBins && !lazy && !split) {
        // this tile's bin arrives unsorted: order it by (depth bits, index) in LDS, keep it there
        // for the staging below and write the sorted indices (and the tile's range) back for the backward pass
        if (tid == 0) ranges[tile] = range;
        if (nslots <= GSR_BLOCK) {          // one key per thread: register sort + merge by counting (the common case of the native loop)
            GSR_T_TICK(0)
            sort_block_keys((tid < nslots) ? bins[range.x + tid] : ~0ull, s_keys);
            overhead += 2;
        } else {
            int npow = 512;
            while (npow < total) npow <<= 1;
            for (int i = tid; i < npow; i += GSR_BLOCK) s_keys[i] = (i < total) ? bins[range.x + i] : ~0ull;
            __syncthreads();
            GSR_T_TICK(0)
            lds_bitonic_sort(s_keys, npow);
            // (measured: a compare-exchange step of the network costs about a seventh of a group of eight composited entries,
            // twice / four times that above 512 / 1024 keys)
            const int lg = 31 - __builtin_clz((unsigned)npow);
            overhead += (lg * (lg + 1) / 2) * max(1, npow >> 9) / 7;
        }
        for (int i = tid; i < total; i += GSR_BLOCK) point_list[range.x + i] = (uint32_t)s_keys[i];
    }
    GSR_T_TICK(1)
    // T > 0: still compositing.  T <= 0: finished (or outside the image); the pixel's transmittance is -T.  With a
    // negative T every later test_T = T (1 - alpha) is negative, i.e. "below 1e-4": the splat is neither blended nor
    // counted, and the kill branch keeps T where it is -- no flag and no second register to carry.
    float T = inside ? 1.0f : 0.f;
    gsr_f32x2 Crg = {0.f, 0.f}, Cbd = {0.f, 0.f};      // accumulated (r, g) and (b, depth)
    const gsr_f32x2 pxy = {pxf, pyf};
    uint32_t last_contributor = 0;
    float zneed = 0.f;        // depth bound of what this pixel had to look at (rounded up to its group of eight)

    // GSR_LIST_EXACT: `consumed` entries of the segment are ordered (and written to point_list) so far; the keys of the
    // current slice sit in s_keys[0, m).  The other modes make one pass with m = total.
    // ---- one segment of a split tile (see SegCtl) ----
    if (LIST == GSR_LIST_BINS && split) {
        __shared__ uint32_t s_sp_fill, s_sp_last;
        __shared__ int s_sp_walk[4];
        const uint32_t first = blockIdx.x - seg;          // block of the tile's segment 0
        const unsigned long long* keys = bins + range.x;
        float* myrec = sg.rec + (size_t)blockIdx.x * (GSR_SEG_REC_Q * GSR_BLOCK);
        const uint32_t pub_word = (sg.epoch << 2) | 1u;
        // (1) the sample every segment of the tile draws alike (sixteen runs of 64 keys spread over the bin, as sample_slice) and
        // this segment's depth range (lo, hi]: pivot j = a depth with j / nseg of the sample at or below it
        uint32_t* s_samp = reinterpret_cast<uint32_t*>(s.a);
        const int nruns = (total + GSR_SAMPLE_RUN - 1) / GSR_SAMPLE_RUN;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int i = tid + GSR_BLOCK * j;
            const int run = i / GSR_SAMPLE_RUN;
            const int pos = ((nruns <= 1024 / GSR_SAMPLE_RUN) ? run : (int)(((long long)run * nruns) / (1024 / GSR_SAMPLE_RUN))) * GSR_SAMPLE_RUN + (i & (GSR_SAMPLE_RUN - 1));
            s_samp[i] = (pos < total) ? (uint32_t)(keys[pos] >> 32) : 0xFFFFFFFFu;
        }
        if (tid == 0) s_sp_fill = 0u;
        __syncthreads();
        uint32_t lo_d = 0u, hi_d = 0xFFFFFFFEu;
        {
            uint32_t v[16];
#pragma unroll
            for (int q = 0; q < 4; q++) {
                const uint4 x = reinterpret_cast<const uint4*>(s_samp)[lane + 64 * q];
                v[4 * q] = x.x; v[4 * q + 1] = x.y; v[4 * q + 2] = x.z; v[4 * q + 3] = x.w;
            }
            int nvalid = 0;
            uint32_t vmin = 0xFFFFFFFFu, vmax = 0u;
#pragma unroll
            for (int q = 0; q < 16; q++) {
                const bool ok = v[q] != 0xFFFFFFFFu;
                nvalid += (int)__popcll(__ballot(ok));
                vmin = min(vmin, v[q]);
                vmax = ok ? max(vmax, v[q]) : vmax;
            }
#pragma unroll
            for (int off = 32; off > 0; off >>= 1) {
                vmin = min(vmin, (uint32_t)__shfl_xor((int)vmin, off, 64));
                vmax = max(vmax, (uint32_t)__shfl_xor((int)vmax, off, 64));
            }
            const uint32_t vmin_u = (uint32_t)__builtin_amdgcn_readfirstlane((int)vmin), vmax_u = (uint32_t)__builtin_amdgcn_readfirstlane((int)vmax);
            // (the tolerance stays below a quarter of the distance between two pivots' ranks, so that consecutive pivots come out in order;
            // the same function of the same data in every wave of every segment: neighbours agree on their common pivot)
            auto pivot = [&](uint32_t j) -> uint32_t {
                const int r = max(1, (int)(((long long)j * nvalid) / (int)nseg));
                const int tol = (nvalid / (int)nseg) >> 2;
                uint32_t lo_b = vmin_u, hi_b = vmax_u;
                while (lo_b < hi_b) {
                    const uint32_t mid = lo_b + ((hi_b - lo_b) >> 1);
                    int c = 0;
#pragma unroll
                    for (int q = 0; q < 16; q++) c += (int)__popcll(__ballot(v[q] <= mid));
                    if (c >= r) { hi_b = mid; if (c <= r + tol) break; }
                    else lo_b = mid + 1u;
                }
                return hi_b;
            };
            if (seg > 0u) lo_d = pivot(seg);
            if (seg + 1u < nseg) hi_d = pivot(seg + 1u);
        }
        GSR_T_COUNT(10, 1000)      // (timing build: marks the rows of split segments)
        GSR_T_TICK(0)
        // (2) one pass over the bin gathers the range's keys (ballot prefix per wave, one LDS atomic per wave and 1 024 keys)
        for (int i0 = 0; i0 < total; i0 += 4 * GSR_BLOCK) {
            unsigned long long k[4];
            bool in[4];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const int i = i0 + j * GSR_BLOCK + tid;
                k[j] = (i < total) ? keys[i] : 0ull;
                const uint32_t d = (uint32_t)(k[j] >> 32);
                in[j] = i < total && (seg == 0u || d > lo_d) && d <= hi_d;
            }
            unsigned long long mk[4];
            uint32_t cnt4 = 0u;
#pragma unroll
            for (int j = 0; j < 4; j++) { mk[j] = __ballot(in[j]); cnt4 += (uint32_t)__popcll(mk[j]); }
            if (cnt4 != 0u) {
                uint32_t at = 0u;
                if (lane == 0) at = atomicAdd(&s_sp_fill, cnt4);
                at = (uint32_t)__builtin_amdgcn_readfirstlane((int)at);
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const uint32_t pos = at + (uint32_t)__popcll(mk[j] & ((1ull << lane) - 1ull));
                    if (in[j] && pos < (uint32_t)GSR_LSORT_CAP) s_keys[pos] = k[j];
                    at += (uint32_t)__popcll(mk[j]);
                }
            }
        }
        __syncthreads();
        int m = (int)s_sp_fill;
        GSR_T_TICK(1)
        if (m > GSR_LSORT_CAP) {
            // (a range beyond the in-LDS sort: thousands of keys at one depth, or a sample far off.  The forward fails -- it is redone --
            // and the tile goes unsplit for a while; this segment carries on as an empty one so that nobody waits for it in vain)
            if (tid == 0) { atomicMax(fail, fail_tag | GSR_FAIL_BOUND); sg.nosplit[tile] = 64u; }
            m = 0;
        }
        if (tid == 0) seg_store_u(&sg.cnt[blockIdx.x], (sg.epoch << 16) | (uint32_t)(m + 1));
        // (3) order
        if (m <= GSR_BLOCK) {
            sort_block_keys((tid < m) ? s_keys[tid] : ~0ull, s_keys);
            overhead += 3;
        } else {
            int npow = 512;
            while (npow < m) npow <<= 1;
            for (int i = m + tid; i < npow; i += GSR_BLOCK) s_keys[i] = ~0ull;
            __syncthreads();
            lds_bitonic_sort(s_keys, npow);
            const int lg = 31 - __builtin_clz((unsigned)npow);
            overhead += 2 + (lg * (lg + 1) / 2) * max(1, npow >> 9) / 7;
        }
        // (4) pass 0: Tl, the product of (1 - alpha) over this pixel's valid entries; pass 1: the walk proper from Ts
        GSR_T_TICK(2)
        const gsr_f32x2 pxy2 = {pxf, pyf};
        const bool one_batch = m <= GSR_BLOCK;      // staged once, kept for both passes
        float Tl = 1.f, Ts = 0.f, Tc = 0.f, Tl2 = 1.f;
        uint32_t basepos = 0u;
        int cntw = 0;
        // (segment 0 knows its Ts -- 1 -- and goes straight to pass 1; the Tl it publishes afterwards is that walk's own chain, or 0 for a
        // pixel that terminated in it: all a later segment needs to know of such a pixel is that it is finished)
        for (int pass = (seg == 0u ? 1 : 0); pass < 2; pass++) {
            if (pass == 1 && seg > 0u) {
                seg_store(&myrec[tid], Tl);
                asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
                __syncthreads();
                if (tid == 0) seg_store_u(&sg.pub[blockIdx.x], pub_word);
                // (every predecessor's publication word, count and product is asked for at once -- a loop of wait-then-load per predecessor
                // is two dependent round trips through L2 for each of up to 31 of them: timing build, S-room-640, 38 k of a median
                // segment's 142 k cycles.  The products are still multiplied in segment order.)
                static_assert(GSR_SEG_MAX <= 64, "one lane per predecessor");
                bool ok = false;
                // (bounded: a forward that gave up waiting fails and the tile goes unsplit for a while.  Round 6: 2^13 polls ~ 10 ms, was 2^21 --
                // seconds per stuck range when many calls share the GPU, see GSR_SPLIT_MAX_CALLS in gsr_api.hip)
                for (uint32_t spins = 0; spins < (1u << 13); spins++) {
                    const bool mine = (uint32_t)lane >= seg || seg_load_u(&sg.pub[first + (uint32_t)lane]) == pub_word;
                    if (__all(mine)) { ok = true; break; }
                    __builtin_amdgcn_s_sleep(8);
                }
                {
                    uint32_t c = ((uint32_t)lane < seg) ? (seg_load_u(&sg.cnt[first + (uint32_t)lane]) & 0xFFFFu) - 1u : 0u;
#pragma unroll
                    for (int off = 32; off > 0; off >>= 1) c += (uint32_t)__shfl_xor((int)c, off, 64);
                    basepos += c;
                }
                float t = inside ? 1.f : 0.f;
                for (uint32_t q0 = 0; q0 < seg; q0 += 8u) {
                    float v[8];
#pragma unroll
                    for (uint32_t j = 0; j < 8u; j++)
                        v[j] = (q0 + j < seg) ? seg_load(&sg.rec[(size_t)(first + q0 + j) * (GSR_SEG_REC_Q * GSR_BLOCK) + tid]) : 1.f;
#pragma unroll
                    for (uint32_t j = 0; j < 8u; j++) t = t * v[j];
                }
                // (never seen; a forward that gave up waiting must not count.  Reported as a failed SPECULATION, with the tile unsplit for the
                // next 64 forwards -- not as a bin overflow, which would send the rest of the call through count -> scan -> emit)
                if (!ok && tid == 0) { atomicMax(fail, fail_tag | GSR_FAIL_BOUND); sg.nosplit[tile] = 64u; }
                GSR_T_TICK(5)
                Ts = t;
                Tc = (t >= 0.0001f) ? t : -t;          // below 1e-4: this pixel terminated in an earlier segment
                if (one_batch && tid < m) {
                    const float4 b4 = s.b[tid];
                    point_list[range.x + basepos + tid] = pack_qm ? (__float_as_uint(b4.z) | (__float_as_uint(b4.w) << 28)) : __float_as_uint(b4.z);
                }
            } else if (pass == 1) {          // segment 0
                Ts = inside ? 1.f : 0.f;
                Tc = Ts;
            }
            for (int base = 0; base < m; base += GSR_BLOCK) {
                if (pass == 1) { if (__syncthreads_and(Tc <= 0.f)) break; }
                else if (base > 0) __syncthreads();
                const int n = min(GSR_BLOCK, m - base);
                if (pass == 0 || !one_batch || seg == 0u) {
                    overhead += 3;
                    if (tid < n) {
                        const uint32_t id = (uint32_t)s_keys[base + tid];
                        const float4* r = reinterpret_cast<const float4*>(rec + (size_t)id * GSR_REC_STRIDE);
                        const float4 r0 = r[0], r1 = r[1], r2 = r[2];
                        const uint32_t qm = quadrant_mask(r0.x, r0.y, r1.x * (-2.0f / GSR_LOG2E), r0.z * (-1.0f / GSR_LOG2E), r0.w * (-2.0f / GSR_LOG2E), r1.y,
                                                          tx * GSR_TILE, ty * GSR_TILE);
                        if (pass == 1) point_list[range.x + basepos + base + tid] = pack_qm ? (id | (qm << 28)) : id;
                        s.a[tid] = r0;
                        s.b[tid] = make_float4(r1.x, r1.y, __uint_as_float(id), __uint_as_float(qm));
                        s.c[tid] = make_float4(r2.x, r2.y, r2.z, r1.z);
                    }
                    __syncthreads();
                    cntw = 0;
                    for (int c0 = 0; c0 < n; c0 += 64) {
                        const int jj = c0 + lane;
                        const bool hit = jj < n && ((__float_as_uint(s.b[min(jj, GSR_BLOCK - 1)].w) >> wv) & 1u);
                        const unsigned long long mk = __ballot(hit);
                        if (hit) s.list[wv][cntw + __popcll(mk & ((1ull << lane) - 1ull))] = (uint8_t)jj;
                        cntw += (int)__popcll(mk);
                    }
                }
                // (the walks: eight entries per step from one 8-byte read of the wave's list, like the unsplit kernel's)
                const int full = cntw & ~7;
                GSR_T_TICK(3)
                if (pass == 0) {
                    auto body0 = [&](int j) {
                        const float4 A = s.a[j];
                        const float2 B = *reinterpret_cast<const float2*>(&s.b[j]);
                        const gsr_f32x2 d = (gsr_f32x2){A.x, A.y} - pxy2;
                        const gsr_f32x2 tu = (gsr_f32x2){A.z, A.w} * (gsr_f32x2){d.y, d.y};
                        const float p2 = __builtin_fmaf(d.x, __builtin_fmaf(B.x, d.x, tu.x), tu.y * d.y);
                        const float G = __builtin_amdgcn_exp2f(p2);
                        const float alpha = fminf(0.99f, B.y * G);
                        const bool valid = !(alpha < 1.0f / 255.0f) && !(p2 > 0.0f);
                        Tl = valid ? Tl * (1.f - alpha) : Tl;
                    };
                    for (int g0 = 0; g0 < full; g0 += 8) {
                        const unsigned long long packed = *reinterpret_cast<const unsigned long long*>(&s.list[wv][g0]);
                        const uint32_t plo = __builtin_amdgcn_readfirstlane((uint32_t)packed);
                        const uint32_t phi = __builtin_amdgcn_readfirstlane((uint32_t)(packed >> 32));
#pragma unroll
                        for (int sidx = 0; sidx < 8; sidx++) body0((int)(((sidx < 4 ? plo : phi) >> (8 * (sidx & 3))) & 0xFFu));
                    }
                    for (int k0 = full; k0 < cntw; k0++) body0(__builtin_amdgcn_readfirstlane((int)s.list[wv][k0]));
                    GSR_T_TICK(4)
                } else {
                    float zlast = 0.f;
                    auto body1 = [&](int j) {
                        const float4 A = s.a[j];
                        const float2 B = *reinterpret_cast<const float2*>(&s.b[j]);
                        const float4 Cc = s.c[j];
                        const gsr_f32x2 d = (gsr_f32x2){A.x, A.y} - pxy2;
                        const gsr_f32x2 tu = (gsr_f32x2){A.z, A.w} * (gsr_f32x2){d.y, d.y};
                        const float p2 = __builtin_fmaf(d.x, __builtin_fmaf(B.x, d.x, tu.x), tu.y * d.y);
                        const float G = __builtin_amdgcn_exp2f(p2);
                        const float alpha = fminf(0.99f, B.y * G);
                        const bool valid = !(alpha < 1.0f / 255.0f) && !(p2 > 0.0f);
                        const float Tln = Tl2 * (1.f - alpha);          // the same chain as pass 0, bit for bit
                        const float test_T = Ts * Tln;
                        const bool alive = Tc > 0.f;
                        const bool kill = valid && alive && test_T < 0.0001f;
                        const bool blend = valid && alive && !kill;
                        const float w = blend ? alpha * Tc : 0.f;
                        Crg = __builtin_elementwise_fma((gsr_f32x2){Cc.x, Cc.y}, (gsr_f32x2){w, w}, Crg);
                        Cbd = __builtin_elementwise_fma((gsr_f32x2){Cc.z, Cc.w}, (gsr_f32x2){w, w}, Cbd);
                        Tc = kill ? -Tc : (blend ? test_T : Tc);
                        Tl2 = valid ? Tln : Tl2;
                        last_contributor = blend ? (uint32_t)(basepos + base + j + 1) : last_contributor;
                        zlast = Cc.w;
                        if (TOUCHED) {      // pose package: pixels where the splat was blended with T still > 0.5 (as the unsplit walk counts them)
                            const int c = (int)__popcll(__ballot(valid && alive && test_T > 0.5f));
                            if (c != 0 && lane == 0) atomicAdd(&n_touched[__float_as_uint(s.b[j].z)], c);
                        }
                    };
                    for (int g0 = 0; g0 < full; g0 += 8) {
                        if (__all(Tc <= 0.f)) break;
                        walked++;
                        const unsigned long long packed = *reinterpret_cast<const unsigned long long*>(&s.list[wv][g0]);
                        const uint32_t plo = __builtin_amdgcn_readfirstlane((uint32_t)packed);
                        const uint32_t phi = __builtin_amdgcn_readfirstlane((uint32_t)(packed >> 32));
                        const bool alive0 = Tc > 0.f;
#pragma unroll
                        for (int sidx = 0; sidx < 8; sidx++) body1((int)(((sidx < 4 ? plo : phi) >> (8 * (sidx & 3))) & 0xFFu));
                        zneed = alive0 ? zlast : zneed;          // (depth needed: rounded up to the group of eight, like the unsplit walk)
                    }
                    for (int k0 = full; k0 < cntw; k0++) {
                        if (__all(Tc <= 0.f)) break;
                        const bool alive0 = Tc > 0.f;
                        body1(__builtin_amdgcn_readfirstlane((int)s.list[wv][k0]));
                        zneed = alive0 ? zlast : zneed;
                    }
                    GSR_T_TICK(6)
                }
            }
        }
        if (seg == 0u) {
            seg_store(&myrec[tid], (Tc > 0.f) ? Tl2 : 0.f);
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            __syncthreads();
            if (tid == 0) seg_store_u(&sg.pub[blockIdx.x], pub_word);
        }
        // the segment's record; then the ticket: who finishes last adds the tile up
        seg_store(&myrec[1 * GSR_BLOCK + tid], Ts);
        seg_store(&myrec[2 * GSR_BLOCK + tid], Tc);
        seg_store(&myrec[3 * GSR_BLOCK + tid], Crg.x);
        seg_store(&myrec[4 * GSR_BLOCK + tid], Crg.y);
        seg_store(&myrec[5 * GSR_BLOCK + tid], Cbd.x);
        seg_store(&myrec[6 * GSR_BLOCK + tid], Cbd.y);
        seg_store(&myrec[7 * GSR_BLOCK + tid], __uint_as_float(last_contributor));
        seg_store(&myrec[8 * GSR_BLOCK + tid], inside ? zneed : 0.f);
        if (lane == 0) s_sp_walk[wv] = walked;
        __syncthreads();
        if (tid == 0) seg_store(&myrec[9 * GSR_BLOCK], (float)(max(max(s_sp_walk[0], s_sp_walk[1]), max(s_sp_walk[2], s_sp_walk[3])) + 1 + overhead));
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        if (tid == 0) {
            const bool last = atomicAdd(&sg.ticket[2 * tile + 1], 1u) == nseg - 1u;
            if (last) sg.ticket[2 * tile + 1] = 0u;
            s_sp_last = last ? 1u : 0u;
        }
        __syncthreads();
        GSR_T_TICK(7)
        if (s_sp_last == 0u) { GSR_T_FLUSH(0) return; }
        {
            float Tfin = inside ? 1.f : 0.f, zn = 0.f, work = 0.f;
            bool dead = false;
            uint32_t lastc = 0u, tot = 0u;
            gsr_f32x2 crg = {0.f, 0.f}, cbd = {0.f, 0.f};
            for (uint32_t q = 0; q < nseg; q++) {
                const float* r = sg.rec + (size_t)(first + q) * (GSR_SEG_REC_Q * GSR_BLOCK);
                const float te = seg_load(r + 2 * GSR_BLOCK + tid);
                if (!dead) { Tfin = te; dead = te <= 0.f; }
                crg += (gsr_f32x2){seg_load(r + 3 * GSR_BLOCK + tid), seg_load(r + 4 * GSR_BLOCK + tid)};
                cbd += (gsr_f32x2){seg_load(r + 5 * GSR_BLOCK + tid), seg_load(r + 6 * GSR_BLOCK + tid)};
                lastc = max(lastc, __float_as_uint(seg_load(r + 7 * GSR_BLOCK + tid)));
                zn = fmaxf(zn, seg_load(r + 8 * GSR_BLOCK + tid));
                work += seg_load(r + 9 * GSR_BLOCK);
                tot += (seg_load_u(&sg.cnt[first + q]) & 0xFFFFu) - 1u;
            }
            T = Tfin; Crg = crg; Cbd = cbd; last_contributor = lastc; zneed = zn;
            walked = (int)work; overhead = 0;
            if (tid == 0) { ranges[tile] = make_uint2(range.x, range.x + tot); if (sg.len != nullptr) sg.len[tile] = tot; }
        }
        GSR_T_TICK(8)
    }
    int consumed = 0, m = total, slice_no = 0;
    unsigned long long slice_lo = 0ull;
  for (bool first_slice = true;; first_slice = false) {
    if (split) break;          // (a split tile's finalising segment: straight to the epilogue)
    if (lazy) {
        if (consumed >= total) break;
        if (__syncthreads_and(T <= 0.f)) break;          // every pixel of the tile has terminated: the rest is never ordered
        const unsigned long long* seg = bins + range.x;
        const int remaining = total - consumed;
        unsigned long long slice_hi = ~0ull;
        // slice sizes: the first aims at a couple of hundred keys (most tiles saturate within it, and up to 256 keys sort in
        // registers); a tile that wants more wants much more
        int want = (slice_no == 0) ? GSR_SLICE_WANT0 : ((slice_no == 1) ? GSR_SLICE_WANT1 : GSR_SLICE_WANT2);
        m = -1;
        for (int attempt = 0; attempt < 3 && m < 0; attempt++) {
            const int got = sample_slice(seg, nslots, first_slice, slice_lo, remaining, want, GSR_LSORT_CAP, reinterpret_cast<uint32_t*>(s.a), s_keys, slice_hi GSR_T_ARGS);
            if (got >= 1 && got <= GSR_LSORT_CAP) m = got;
            else if (got == 0) break;                                      // the sampled front of the segment is used up
            else { want = max(16, want >> 2); __syncthreads(); }          // too many at or below the threshold: a smaller share
        }
        if (m < 0) {
            // thousands of keys at one depth, or nothing left in the sampled front of the segment: exact radix selection
            m = remaining;
            slice_hi = ~0ull;
            if (remaining > GSR_LSORT_CAP)
                select_slice(seg, nslots, first_slice, slice_lo, GSR_LSORT_CAP, reinterpret_cast<uint32_t*>(s_keys), slice_hi, m);
            if (m <= 0) {          // cannot happen with distinct keys (the index is part of them): corrupted bins -- fail loudly, never spin
                if (tid == 0) atomicMax(fail, fail_tag | GSR_FAIL_OVERFLOW);
                break;
            }
            __shared__ uint32_t s_fill2;
            if (tid == 0) s_fill2 = 0u;
            __syncthreads();
            for (int i = tid; i < nslots; i += GSR_BLOCK) {
                const unsigned long long k = seg[i];
                if ((first_slice || k > slice_lo) && k <= slice_hi && k != ~0ull) s_keys[atomicAdd(&s_fill2, 1u)] = k;
            }
            __syncthreads();
        }
        slice_no++;
        if (m <= GSR_BLOCK) {
            sort_block_keys((tid < m) ? s_keys[tid] : ~0ull, s_keys);
            overhead += 3;
        } else {
            int npow = 512;
            while (npow < m) npow <<= 1;
            for (int i = m + tid; i < npow; i += GSR_BLOCK) s_keys[i] = ~0ull;
            __syncthreads();
            lds_bitonic_sort(s_keys, npow);
            const int lg = 31 - __builtin_clz((unsigned)npow);
            overhead += 2 + (lg * (lg + 1) / 2) * max(1, npow >> 9) / 7;
        }
        GSR_T_TICK_O(7)
        for (int i = tid; i < m; i += GSR_BLOCK) point_list[range.x + consumed + i] = (uint32_t)s_keys[i];
        slice_lo = slice_hi;
    }
    for (int base = 0; base < m; base += GSR_BLOCK) {
        if (__syncthreads_and(T <= 0.f)) break;
        GSR_T_TICK(2)
        GSR_T_COUNT(10, 1)
        const int n = min(GSR_BLOCK, m - base);
        overhead += 3;
        {
            const bool have = tid < n;
            uint32_t id = 0u;
            float4 r0 = make_float4(0.f, 0.f, 0.f, 0.f), r1 = r0, r2 = r0;
            if (have) {
                id = (LIST != GSR_LIST_SORTED) ? (uint32_t)s_keys[base + tid]
                                                : (pack_qm ? (point_list[range.x + base + tid] & 0x0FFFFFFFu) : point_list[range.x + base + tid]);
                const float4* r = reinterpret_cast<const float4*>(rec + (size_t)id * GSR_REC_STRIDE);
                r0 = r[0]; r1 = r[1];
                if (kFull && lz.shs != nullptr) {
                    // (LazySH: another workgroup of this launch may be publishing this quad right now.  It is read and written as ONE
                    // 16-byte access -- a volatile vector access, which the compiler neither splits nor reorders nor repeats; on gfx950 an
                    // aligned global_load / store_dwordx4 is a single transaction on one cache line, so a reader sees either the
                    // unevaluated quad (w = 0) or the complete one (w = 1).  Two tiles that both find w = 0 both evaluate the colour and
                    // store the same bits; the same goes for the byte they store into `clamped`.)
                    const gsr_f32x4 q = *reinterpret_cast<const volatile gsr_f32x4*>(r + 2);
                    r2 = make_float4(q[0], q[1], q[2], q[3]);
                } else r2 = r[2];
            }
#if GSR_TIMING
            if (kFull) { asm volatile("" :: "v"(r0.x), "v"(r1.x), "v"(r2.w)); GSR_T_TICK(0) }
#endif
            if (kFull && lz.shs != nullptr) {          // first tile to stage a splat: its colour (LazySH)
                const bool need = have && r2.w == 0.f;
                // (measured in round 4: taking the lanes that need a colour sixteen at a time, their rows as coalesced streams through an
                // LDS slab, one channel of one row per lane -- TWICE as slow, 55 k against 25 k cycles per wave: the phase is a chain of
                // memory round trips of ~8 k cycles each while every tile of the image stages at the same time, and the chunks add
                // round trips; the per-lane row loads below put all of them in flight at once)
                if (need) {
                    uint8_t cb;
                    const float3 pm = make_float3(lz.means[3 * (size_t)id], lz.means[3 * (size_t)id + 1], lz.means[3 * (size_t)id + 2]);
                    const float3 c = sh16_vector_ok(lz.M, lz.shs)
                                         ? sh_row16_to_rgb(lz.D, pm, lz.campos, reinterpret_cast<const float4*>(lz.shs) + (size_t)id * GSR_SH16_ROW4, cb)
                                         : sh_to_rgb(lz.D, lz.M, pm, lz.campos, lz.shs + (size_t)id * lz.M * 3, cb);
                    r2 = make_float4(c.x, c.y, c.z, 1.f);
                    *reinterpret_cast<volatile gsr_f32x4*>(lz.rec + (size_t)id * GSR_REC_STRIDE + 8) = (gsr_f32x4){c.x, c.y, c.z, 1.f};
                    lz.clamped[id] = cb;
                }
            }
#if GSR_TIMING
            if (kFull) { GSR_T_TICK(1) }
#endif
            if (have) {
                const uint32_t qm = quadrant_mask(r0.x, r0.y, r1.x * (-2.0f / GSR_LOG2E), r0.z * (-1.0f / GSR_LOG2E), r0.w * (-2.0f / GSR_LOG2E), r1.y,
                                                  tx * GSR_TILE, ty * GSR_TILE);
                if (LIST != GSR_LIST_SORTED && pack_qm) point_list[range.x + consumed + base + tid] = id | (qm << 28);
                s.a[tid] = r0;
                s.b[tid] = make_float4(r1.x, r1.y, __uint_as_float(id), __uint_as_float(qm));
                s.c[tid] = make_float4(r2.x, r2.y, r2.z, r1.z);
            }
        }
        __syncthreads();
        GSR_T_TICK(3)
        // this wave's compacted list (order preserved)
        int cnt = 0;
        for (int c0 = 0; c0 < n; c0 += 64) {
            const int jj = c0 + lane;
            const bool hit = jj < n && ((__float_as_uint(s.b[min(jj, GSR_BLOCK - 1)].w) >> wv) & 1u);
            const unsigned long long mk = __ballot(hit);
            if (hit) s.list[wv][cnt + __popcll(mk & ((1ull << lane) - 1ull))] = (uint8_t)jj;
            cnt += (int)__popcll(mk);
        }
        GSR_T_TICK(GSR_TO(4))
        const int full = cnt & ~7;
        for (int g0 = 0; g0 < full; g0 += 8) {
            if (__all(T <= 0.f)) break;                // whole wave finished: stop early
            walked++;
            GSR_T_COUNT(11, 8)
            const unsigned long long packed = *reinterpret_cast<const unsigned long long*>(&s.list[wv][g0]);
            const uint32_t plo = __builtin_amdgcn_readfirstlane((uint32_t)packed);
            const uint32_t phi = __builtin_amdgcn_readfirstlane((uint32_t)(packed >> 32));
            const bool alive0 = T > 0.f;
            float zlast = 0.f;
            int tcnt = 0;              // n_touched: lane k of the wave ends up with the count of the group's k-th splat
#pragma unroll
            for (int sidx = 0; sidx < 8; sidx++) {
                const int j = (int)(((sidx < 4 ? plo : phi) >> (8 * (sidx & 3))) & 0xFFu);
                const float4 A = s.a[j];
                const float2 B = *reinterpret_cast<const float2*>(&s.b[j]);
                const float4 Cc = s.c[j];
                const gsr_f32x2 d = (gsr_f32x2){A.x, A.y} - pxy;                      // dx, dy
                const gsr_f32x2 tu = (gsr_f32x2){A.z, A.w} * (gsr_f32x2){d.y, d.y};   // B2 dy, C2 dy
                const float p2 = __builtin_fmaf(d.x, __builtin_fmaf(B.x, d.x, tu.x), tu.y * d.y);
                const float G = __builtin_amdgcn_exp2f(p2);
                const float alpha = fminf(0.99f, B.y * G);
                const float test_T = T * (1.f - alpha);
                const bool valid = !(alpha < 1.0f / 255.0f) && !(p2 > 0.0f) &&      // power > 0: skipped (forward.cu:342)
                                   (!RECOUNT || (uint32_t)(consumed + base + j + 1) <= rc_lim);
                const bool kill = !RECOUNT && valid && test_T < 0.0001f;
                const bool blend = valid && !kill;
                const float w = blend ? alpha * T : 0.f;
                Crg = __builtin_elementwise_fma((gsr_f32x2){Cc.x, Cc.y}, (gsr_f32x2){w, w}, Crg);
                Cbd = __builtin_elementwise_fma((gsr_f32x2){Cc.z, Cc.w}, (gsr_f32x2){w, w}, Cbd);
                T = kill ? __uint_as_float(__float_as_uint(T) | 0x80000000u) : (valid ? test_T : T);      // kill: T -> -|T|
                last_contributor = blend ? (uint32_t)(consumed + base + j + 1) : last_contributor;      // 1-based position in the tile list
#if GSR_TIMING
                (void)alive0;
#endif
                if (TOUCHED) {
                    // pose package: count pixels where the splat was blended with T still > 0.5
                    const int c = (int)__popcll(__ballot(valid && test_T > 0.5f));
                    asm volatile("v_writelane_b32 %0, %1, %2" : "+v"(tcnt) : "s"(c), "i"(sidx));
                }
                if (sidx == 7) zlast = Cc.w;
            }
            zneed = alive0 ? zlast : zneed;
            if (TOUCHED) {
                if (lane < 8 && tcnt != 0) {
                    const int j = (int)s.list[wv][g0 + lane];
                    atomicAdd(&n_touched[__float_as_uint(s.b[j].z)], tcnt);
                }
            }
        }
        // tail: fewer than eight entries left in this wave's list
        for (int k = full; k < cnt; k++) {
            if (__all(T <= 0.f)) break;
            GSR_T_COUNT(11, 1)
            const int j = __builtin_amdgcn_readfirstlane((int)s.list[wv][k]);
            const float4 A = s.a[j];
            const float4 B = s.b[j];
            const float4 Cc = s.c[j];
            if (T > 0.f) zneed = Cc.w;
            const gsr_f32x2 d = (gsr_f32x2){A.x, A.y} - pxy;
            const gsr_f32x2 tu = (gsr_f32x2){A.z, A.w} * (gsr_f32x2){d.y, d.y};
            const float p2 = __builtin_fmaf(d.x, __builtin_fmaf(B.x, d.x, tu.x), tu.y * d.y);
            const float G = __builtin_amdgcn_exp2f(p2);
            const float alpha = fminf(0.99f, B.y * G);
            const float test_T = T * (1.f - alpha);
            const bool valid = !(alpha < 1.0f / 255.0f) && !(p2 > 0.0f) && (!RECOUNT || (uint32_t)(consumed + base + j + 1) <= rc_lim);
            const bool kill = !RECOUNT && valid && test_T < 0.0001f;
            const bool blend = valid && !kill;
            const float w = blend ? alpha * T : 0.f;
            Crg = __builtin_elementwise_fma((gsr_f32x2){Cc.x, Cc.y}, (gsr_f32x2){w, w}, Crg);
            Cbd = __builtin_elementwise_fma((gsr_f32x2){Cc.z, Cc.w}, (gsr_f32x2){w, w}, Cbd);
            T = kill ? __uint_as_float(__float_as_uint(T) | 0x80000000u) : (valid ? test_T : T);
            last_contributor = blend ? (uint32_t)(consumed + base + j + 1) : last_contributor;
            if (TOUCHED) {
                const int c = (int)__popcll(__ballot(valid && test_T > 0.5f));
                if (c != 0 && lane == 0) atomicAdd(&n_touched[__float_as_uint(B.z)], c);
            }
        }
        GSR_T_TICK(5)
    }
    if (!lazy) break;
    consumed += m;
    __syncthreads();          // (the next slice overwrites s_keys and the staging buffers)
  }
    if (RECOUNT) return;          // (the images, n_contrib, the bounds: all as the forward left them)
    // GSR_LIST_EXACT: the tile's range is what has been ORDERED -- all that the backward pass and a re-compositing of
    // these lists (n_touched) can need: no pixel looks beyond the slice in which the last one terminated
    if (lazy && tid == 0) ranges[tile] = make_uint2(range.x, range.x + (uint32_t)min(consumed, total));
    if (sg.len != nullptr && !split && tid == 0) sg.len[tile] = (uint32_t)(lazy ? min(consumed, total) : total);
    GSR_T_TICK(GSR_TO(6))
    if (tile_work != nullptr) {      // this tile's weight in the next iteration's launch order
        __shared__ int s_walk[4];
        if (lane == 0) s_walk[wv] = walked;
        __syncthreads();
        if (tid == 0) tile_work[tile] = (uint32_t)(max(max(s_walk[0], s_walk[1]), max(s_walk[2], s_walk[3])) + 1 + overhead);
    }
    const bool done = (T <= 0.f);
    const float T_out = fabsf(T);
    if (zb_next != nullptr) {
        // Native loop bookkeeping: how deep did this tile have to look?  Next iteration's binning drops what
        // lies behind that (plus a margin); if a pixel is still unsaturated at the end of a list from which
        // entries were dropped, the speculation failed and the host redoes this forward with full lists.
#if GSR_TIMING
        const long long t_bar0_ = clock64();
#endif
        const int unfinished = __syncthreads_or(inside && !done);
#if GSR_TIMING
        GSR_T_COUNT(8, clock64() - t_bar0_)      // slot 8: cycles this wave waited for the tile's other waves at the end of its walk
#endif
        float zm = inside ? zneed : 0.f;
#pragma unroll
        for (int off = 32; off > 0; off >>= 1) zm = fmaxf(zm, __shfl_xor(zm, off, 64));
        if (lane == 0) s_zmax[wv] = zm;
        __syncthreads();
        if (tid == 0) {
            zm = fmaxf(fmaxf(s_zmax[0], s_zmax[1]), fmaxf(s_zmax[2], s_zmax[3]));
            float bound = unfinished ? __builtin_huge_valf() : zm;      // (the margin is applied where the bound is used)
            const bool failed_here = unfinished && zb_used != nullptr && zb_used[tile] < __builtin_huge_valf();
            if (tile_hold != nullptr) {
                // A tile at the edge of the map's coverage saturates in one iteration and not in the next: with a bound recorded every
                // time it saturates it fails every other forward (measured on poses 0.3 m / 10 deg off the map's reference view: 33
                // failed groups in a 50-iteration refinement).  A tile that failed TWICE in a call keeps its complete list for the next
                // GSR_HOLD_FORWARDS forwards -- its own list only; everybody else keeps speculating.
                // (the FIRST failure of a tile in a call is not held -- hold_after = 2: a warm start from another frame's bounds fails in many
                // tiles once, and their retry records good bounds; holding at the first failure was measured in round 5: nothing gained on
                // S-room-640, and a held tile in front of a dense object overflows its bin)
                const uint32_t word = tile_hold[tile];
                uint32_t hold = word & 0xFFu, nfail = word >> 8;
                // (a tile that keeps failing is left alone for longer each time: 32, 64, 128, 255 forwards)
                if (failed_here) {
                    nfail = (nfail < 0xFFFFu) ? nfail + 1u : nfail;
                    hold = 0u;
                    if (nfail >= sg.hold_after) { const uint32_t k = nfail - sg.hold_after; hold = (k >= 3u) ? 255u : (GSR_HOLD_FORWARDS << k); }
                }
                else if (hold > 0u) hold--;
                if (failed_here || (word & 0xFFu) != 0u) tile_hold[tile] = (nfail << 8) | hold;
                if (hold > 0u) bound = __builtin_huge_valf();
            }
            zb_next[tile] = bound;
            const int sb = (ty >> 2) * sbx + (tx >> 2);
            atomicMax(reinterpret_cast<int*>(zbc_next) + sb, __float_as_int(bound));     // bounds are >= 0: int order = float order
            // zb_used: the bounds this forward was binned with.  Instances can only have been dropped from a tile whose
            // bound was finite; if such a tile ends with an unsaturated pixel, a dropped instance may be missing.
            if (failed_here) atomicMax(fail, fail_tag | GSR_FAIL_BOUND);
        }
    }
    const size_t N = (size_t)W * H;
    const float Dd = Cbd.y;
    const float img3[3] = {Crg.x + T_out * bg[0], Crg.y + T_out * bg[1], Cbd.x + T_out * bg[2]};
    if (inside) {
        n_contrib[pix_id] = last_contributor;
        out_color[pix_id] = img3[0];
        out_color[N + pix_id] = img3[1];
        out_color[2 * N + pix_id] = img3[2];
        out_alpha[pix_id] = 1.f - T_out;
        out_depth[pix_id] = Dd;
    }
    if (fl.out != nullptr && !(fl.conv != nullptr && *fl.conv != 0.f)) {
        // fused tracking loss: same arithmetic as k_tracking_loss, on the values just written
        __shared__ float s_red[4][3];
        const float ea = expf(fl.exposure[0]), eb = fl.exposure[1];
        const float inv3n = 1.f / (3.f * (float)N), invn = 1.f / (float)N;
        float l = 0.f, da = 0.f, db = 0.f;
        if (inside) {
            const bool om = (1.f - T_out) > fl.opacity_thr;
            const float gm = fl.grad_mask[pix_id] ? 1.f : 0.f;
            const float w = om ? gm : 0.f;
#pragma unroll
            for (int c = 0; c < 3; c++) {
                const float img = img3[c];
                const float d = (ea * img + eb) * gm - fl.gt_image[(size_t)c * N + pix_id] * gm;
                if (om) l += fabsf(d) * inv3n;
                const float g = w * sgnf(d) * inv3n;
                fl.dL_dimage[(size_t)c * N + pix_id] = g * ea;
                da += g * ea * img;
                db += g;
            }
            float gdp = 0.f;
            if (!fl.monocular) {
                const float gd = fl.gt_depth[pix_id];
                const float dm = (gd > 0.01f && om) ? gm : 0.f;
                const float dd = Dd * dm - gd * dm;
                l += fl.depth_w * fabsf(dd) * invn;
                gdp = fl.depth_w * dm * sgnf(dd) * invn;
            }
            fl.dL_ddepth[pix_id] = gdp;
        }
        l = wave_sum(l); da = wave_sum(da); db = wave_sum(db);
        if (lane == 0) { s_red[wv][0] = l; s_red[wv][1] = da; s_red[wv][2] = db; }
        __syncthreads();
        if (tid < 3) {
            const float t = s_red[0][tid] + s_red[1][tid] + s_red[2][tid] + s_red[3][tid];
            float* shard = fl.out + (blockIdx.x & (GSR_LOSS_SHARDS - 1)) * 16;      // (fl.out: this group's buffer, see PoseStepArgs::loss_shards)
            if (t != 0.f) {
                // (deterministic option; word 3 of the shard counts non-finite sums: the pose step then reports NaN, as float sums would)
                if (fl.det) atomicAdd(reinterpret_cast<unsigned long long*>(shard) + (__builtin_isfinite(t) ? tid : 3),
                                      __builtin_isfinite(t) ? (unsigned long long)to_fixed(t, GSR_FIX_LOSS) : 1ull);
                else atomicAdd(&shard[tid], t);
            }
        }
    }
    GSR_T_TICK(GSR_TO(7))
    GSR_T_FLUSH(0)
}

// ---------------------------------------------------------------------------------------------
// K7  per-tile back-to-front gradient (replaces backward.cu:399-581 renderCUDA).
// Same tile / lane mapping as K6.  Differences from the reference's schedule (results identical up to fp32
// summation order):  (1) the walk starts at the tile's deepest contributor (max n_contrib), not at the end of
// the tile list;  (2) the per-splat sums are contracted over the 64 pixels of a wave on the matrix cores, written to
// per-wave slices in LDS, added up once per batch, and leave the workgroup as ONE global atomic per (tile, splat,
// quantity) instead of one per (pixel, splat, quantity);  (3) a list entry's splat record is read with scalar loads
// (GSR_REC_*), not staged in LDS.
// ---------------------------------------------------------------------------------------------
// packed per-Gaussian accumulator record of K7 (floats): 0-2 dL/dcolor, 3-4 dL/dmean2D, 5-7 dL/dconic (a,b,c),
// 8 dL/dopacity, 9 dL/dz (pose package), 10-11 padding
#define GSR_ACC_STRIDE 12
// Each (pixel, splat) pair only produces TWO weights,
//     W1 = alpha * T                      (d pixel / d colour_i,  backward.cu:517)
//     W2 = G * dL/d(alpha_i)              (backward.cu:549-578 before the per-quantity factors)
// and every per-splat gradient sum is a pixel moment of them:
//     dL/dcolour = sum W1 (dpx,dpy,dpz)     dL/dz = sum W1 dL_ddepth      dL/dopacity = sum W2
//     dL/dmean2D, dL/dconic = o * polynomials in (mu,mv) of  sum W2 (1, u, v, uu, uv, vv)
// with (u,v) the pixel position relative to the tile centre and (mu,mv) the splat mean in the same frame.
// That is a dense contraction  S[splat][col] = sum_pixel W[splat][pixel] * g[pixel][col]  (10 columns), which
// goes to the matrix cores: v_mfma_f32_16x16x4_f32 (exact fp32 FMA chain, MI355X_MICROARCH.md) with
// A = 8 splats x {W1,W2} (16 rows) by 4 pixels, B = 4 pixels by 16 columns, 16 steps per 64-pixel wave.
// The weights are transposed through a per-wave LDS buffer (GSR_WT_REGION below); the 16 B operands per lane are pixel
// constants and stay in registers for the whole kernel.
//
// Like K6 the walk is a dependent chain whose length is (entries) x (instructions per entry), so the per-entry
// body is branch-free: a splat that is skipped for this pixel (behind its last contributor, alpha < 1/255 or
// power > 0) is given alpha = 0, for which every recurrence below is the identity -- T/(1-0) = T, the
// "colour behind" accumulators absorb the previous splat exactly as they would one step later -- instead of
// being branched around.  alpha is recomputed with K6's expression (pre-scaled conic, v_exp_f32), bit for bit.
// ---------------------------------------------------------------------------------------------
template <bool B> struct BoolTag { static constexpr bool value = B; };
#define GSR_WT_STRIDE 17
// Weight transposition for the contraction.  A pixel lane p produces 16 values per group of eight splats (row m = 2 * splat +
// {0: W1, 1: W2}); the MFMA's A operand wants lane (k = lane / 16, m = lane % 16) to hold row m of pixel 4 t + k for the steps
// t = 0 ... 15.  Layout (floats): region k = p % 4 (GSR_WT_REGION apart), inside it row m at 16 m, inside the row the sixteen
// t = p / 4 in four chunks of four with chunk index (t / 4) ^ (m / 4):
//   * a reader fetches its sixteen operands with FOUR ds_read_b128 (one per chunk) in front of sixteen back-to-back MFMAs --
//     the [pixel][17] layout needed sixteen 4-byte reads, each one an LDS round trip in front of an MFMA pair;
//   * region stride 272 = 16 mod 64 and the chunk swizzle make the writers' 64 lanes (fixed m) and each 16-lane reader
//     group (fixed k and chunk) fall into distinct banks;
//   * W1 and W2 of a splat share a chunk swizzle (same m / 4): one ds_write2_b32 per splat, as before.
#define GSR_WT_REGION 272
#define GSR_BWD_STAGE 128      // splats looked at per batch
#define GSR_BWD_LIST 64        // ... of which a wave can take this many onto its list: the batch ends where the first list is full
struct BwdMfmaLDS {
    // (what the WALK reads per entry comes from the packed records in global memory through scalar loads, GSR_REC_*; a padded
    // list entry points at record P, the NULL splat -- opacity 0, so alpha = 0 and every update of the walk is the identity --
    // so that the bodies of a group need no "is there an entry" test)
    uint32_t ids[GSR_BWD_STAGE];             // staged splats, deepest first
    uint8_t qm[GSR_BWD_STAGE];               // their quadrant masks
    uint8_t inv[4][GSR_BWD_STAGE];           // per wave: where on its list a staged splat sits (valid for the ones that are on it)
    uint32_t off[4][GSR_BWD_LIST];           // per wave: record offsets (floats) of its list entries
    alignas(8) uint8_t list[4][GSR_BWD_LIST];   // ... and their staged slots
    // per wave and LIST POSITION: 0-3 = sum W1 (dpx,dpy,dpz,dLd), 4-9 = W2 moments.  Every wave has its own slice and writes each
    // (entry, column) once per batch with a plain store; the recombination adds the slices of the waves that had the splat on
    // their list.  (One shared slice merged with ds_add_f32 cost 123 LDS cycles per instruction -- a float atomic occupies the
    // LDS about three cycles per lane -- two thirds of the kernel's LDS time and 9 of its 60 us.)  Four slices of 128 rows would
    // not fit five workgroups per CU; 64 rows do, and a batch looks at up to 128 splats but ends where the first wave's list is
    // full (a wave takes about half of a tile's splats): 1.2 batches per tile instead of 2, each with its barriers and staging.
    float acc[4][GSR_BWD_LIST][10];
    // per wave: the weight transposition buffer of the contraction, see GSR_WT_REGION (before the walk: [pixel][17] scratch
    // for the B operands, the same 1088 floats; between a batch's walk and the next: the recombined sums on their way out)
    alignas(16) float wt[4][64 * GSR_WT_STRIDE];
    int wmax[4], lim[4];
};

template <bool POSE>
__global__ void __launch_bounds__(GSR_BLOCK, 5) k_render_bwd_mfma(const uint2* __restrict__ ranges,
                                                               const uint32_t* __restrict__ point_list, int W, int H, int gx,
                                                               int ntiles, const float* __restrict__ bg,
                                                               const float* __restrict__ alphas, const uint32_t* __restrict__ n_contrib,
                                                               const float* __restrict__ dL_dpix, const float* __restrict__ dL_ddepths,
                                                               const float* __restrict__ dL_dalphas, float* __restrict__ acc,
                                                               LoopGuard guard, const uint32_t* __restrict__ tile_order,
                                                               uint32_t* __restrict__ tile_work, const float* __restrict__ rec, int P, int pack_qm, int det,
                                                               uint8_t* __restrict__ aflag, SegCtl sg, SegBuild sb)
{
    // (aflag, 2 P bytes: [id] = some tile added to this Gaussian's record, [P + id] = ... to its colour sums.  Idempotent plain
    // byte stores -- every writer stores 1 -- that tell the chain-rule kernel which of the forward's survivors have anything to do,
    // without its reading every survivor's 48-byte record: on complete lists nine survivors in ten were never blended.)
    __shared__ BwdMfmaLDS s;
    const GSR_CONST_AS float* crec = (const GSR_CONST_AS float*)rec;      // (constant address space + wave-uniform offsets: s_load)
    // (the extra workgroup is block 0, everybody else's number is blockIdx.x - 1: dispatched first, its serial chain -- order, list, bounds --
    // runs next to the whole launch.  As the LAST block it started only when a slot came free, i.e. after the first round of tiles on an
    // image with more tiles than resident workgroups, and the launch ended that much later: S-3M-cam 852x480 / 1024x576, K7 68 -> 86 /
    // 78 -> 106 us)
    const uint32_t bid = blockIdx.x - (sb.list != nullptr ? 1u : 0u);
    if (sb.list != nullptr && blockIdx.x == 0u) {          // (also on a frozen iteration: its retry runs the list)
        __shared__ uint32_t s_cls2[GSR_BLOCK];
        tile_order_from_work(sb.work, sb.order, sb.ntiles, s_cls2);
        __syncthreads();
        seg_list_build(sb.work, sb.order, sb.list, sb.nosplit, sb.ntiles, sb.budget, sb.len, sb.host_total, sb.split_ok != 0);
        if (sb.zb != nullptr) {
            __syncthreads();
            dilate_bounds(sb, reinterpret_cast<float*>(sb.order));      // (the order array has served its purpose)
        }
        return;
    }
    if (guard.frozen()) return;
    GSR_T_DECL
    // (sg.list: the forward's launch list, see SegCtl -- a split tile's segments are walked by as many workgroups, each over its own
    // window [lo_pos, hi_pos) of the tile's ordered list, back to front, started from what the forward's records say about the
    // window's far end)
    int tile;
    uint32_t seg = 0u, nseg = 1u;
    if (sg.list != nullptr) {
        const uint32_t e = sg.list[bid];
        if (e == 0xFFFFFFFFu) return;
        tile = (int)(e & 0xFFFFu); seg = (e >> 16) & 0xFFu; nseg = e >> 24;
    } else tile = tile_order ? (int)tile_order[bid] : xcd_remap((int)bid, ntiles);
    const uint32_t first = bid - seg;
    uint32_t lo_pos = 0u, hi_pos = 0x7FFFFFFFu, seg_end = seg + 1u;      // (seg_end: one past the last forward segment of this workgroup's window)
    if (nseg > 1u) {
        if ((sg.cnt[first] & 0xFFFFu) == 0u) {          // the forward did not split this tile after all: segment 0 has all of it
            if (seg != 0u) return;
            nseg = 1u;
        } else {
            // (this kernel's per-workgroup costs -- pixel gradients in, B operands, a recombination per batch -- want longer windows than the
            // forward's one-batch segments: a workgroup takes GSR_BWD_SEG_MERGE consecutive segments, the others leave)
            if (seg % GSR_BWD_SEG_MERGE != 0u) return;
            for (uint32_t q = 0; q < seg; q++) lo_pos += (sg.cnt[first + q] & 0xFFFFu) - 1u;
            hi_pos = lo_pos;
            seg_end = min(seg + GSR_BWD_SEG_MERGE, nseg);
            for (uint32_t q = seg; q < seg_end; q++) hi_pos += (sg.cnt[first + q] & 0xFFFFu) - 1u;
        }
    }
    const int tx = tile % gx, ty = tile / gx;
    const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
    const int px = tx * GSR_TILE + (wv & 1) * 8 + (tid & 7), py = ty * GSR_TILE + (wv >> 1) * 8 + ((tid >> 3) & 7);
    const bool inside = px < W && py < H;
    const int pix_id = W * py + px;
    const float pxf = (float)px, pyf = (float)py;
    const gsr_f32x2 pxy = {pxf, pyf};
    const uint2 range = ranges[tile];
    const size_t N = (size_t)W * H;
    // tile-centred frame for the moments (|u|,|v| <= 7.5 keeps the polynomial recombination well conditioned)
    const float cx0 = (float)(tx * GSR_TILE) + 7.5f, cy0 = (float)(ty * GSR_TILE) + 7.5f;

    const float T_final = inside ? (1.f - alphas[pix_id]) : 0.f;
    float T = T_final;
    float dpx = 0.f, dpy = 0.f, dpz = 0.f, dLd = 0.f, dLa = 0.f;
    if (inside) {
        dpx = dL_dpix[pix_id]; dpy = dL_dpix[N + pix_id]; dpz = dL_dpix[2 * N + pix_id];
        dLd = dL_ddepths[pix_id]; dLa = dL_dalphas[pix_id];
    }
    // Round 6: a pixel whose five incoming gradients are all zero -- outside the frame's gradient mask, or not opaque enough for the
    // tracking loss (descent_utils.py:100-101,118-121: more than half of the pixels under the reference's masks) -- adds exactly
    // nothing to any sum below: every term is linear in (dpx, dpy, dpz, dLd, dLa).  It is treated as a pixel without contributors,
    // so an 8 x 8 block (a wave) or a tile of such pixels walks nothing, and a wave's walk is as long as its deepest LIVE pixel needs.
#ifdef GSR_NO_DEAD_PIXEL_SKIP          // (diagnostic builds: the A/B of this shortcut, HISTORY.md round 6)
    const bool live = inside;
#else
    const bool live = inside && (dpx != 0.f || dpy != 0.f || dpz != 0.f || dLd != 0.f || dLa != 0.f);
#endif
    const int last_contributor = live ? (int)n_contrib[pix_id] : 0;
    const float bg_dot = bg[0] * dpx + bg[1] * dpy + bg[2] * dpz;
    const float nTf_bg = -T_final * bg_dot;

    // B operands: lane (k = lane>>4, j = lane&15) needs g[pixel 4t+k][column j] for t = 0..15
    float* wt = s.wt[wv];
    {
        const float u = pxf - cx0, v = pyf - cy0;
        float* row = wt + lane * GSR_WT_STRIDE;
        row[0] = dpx; row[1] = dpy; row[2] = dpz; row[3] = POSE ? dLd : 0.f;
        row[4] = 1.f; row[5] = u; row[6] = v; row[7] = u * u; row[8] = u * v; row[9] = v * v;
        row[10] = 0.f; row[11] = 0.f; row[12] = 0.f; row[13] = 0.f; row[14] = 0.f; row[15] = 0.f;
    }
    float Breg[16];
#pragma unroll
    for (int t = 0; t < 16; t++) Breg[t] = wt[(4 * t + (lane >> 4)) * GSR_WT_STRIDE + (lane & 15)];

    int m = last_contributor;
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) m = max(m, __shfl_xor(m, off, 64));
    if (lane == 0) s.wmax[wv] = m;
    __syncthreads();
    // (total: one past the deepest list position this workgroup has to look at -- the tile's deepest contributor, or the end of its window)
    const int total = min(max(max(s.wmax[0], s.wmax[1]), max(s.wmax[2], s.wmax[3])), (int)hi_pos);
    const int wave_max = s.wmax[wv];
    if (total <= (int)lo_pos) return;          // (a window behind everything the tile's pixels needed; block-uniform)

    float av = 0.f, lv = 0.f, last_alpha = 0.f, om_last = 1.f;      // the "composited behind me" recurrence, see the loop body (om_last = 1 - last_alpha)
    if (nseg > 1u && seg_end < nseg && inside && (uint32_t)last_contributor > hi_pos) {
        // this pixel goes on behind the window: its transmittance at the window's far end is the next segment's Ts, and what lies behind,
        // composited as seen from there, is (the later segments' sums) / Ts -- for the value v = colour . dL/dpixel + depth dL/ddepth - dL/dalpha
        // the walk's recurrence carries (k_render_fwd's records, see SegCtl)
        const size_t rs = (size_t)GSR_SEG_REC_Q * GSR_BLOCK;
        const float Tb = sg.rec[(size_t)(first + seg_end) * rs + 1 * GSR_BLOCK + tid];
        double cr = 0.0, cg = 0.0, cb = 0.0, cd = 0.0;
        for (uint32_t q = seg_end; q < nseg; q++) {
            const float* r = sg.rec + (size_t)(first + q) * rs;
            cr += r[3 * GSR_BLOCK + tid]; cg += r[4 * GSR_BLOCK + tid]; cb += r[5 * GSR_BLOCK + tid]; cd += r[6 * GSR_BLOCK + tid];
        }
        T = Tb;
        // (in double: one value carries the whole window's "behind" -- the sum's cancellations would otherwise be its error)
        av = (float)((((double)dpx * cr + (double)dpy * cg) + ((double)dpz * cb + (double)dLd * cd)) / (double)Tb - (double)dLa * (1.0 - (double)T_final / (double)Tb));
    }
    const bool simple = __all(dLa == 0.f && nTf_bg == 0.f) != 0;
    int walked = 0;                                  // groups of eight list entries this wave has gone through (-> tile_work)
    const float ddelx_dx = 0.5f * W, ddely_dy = 0.5f * H;
    const int arow = (lane >> 4), acol = (lane & 15);
    // D of the MFMA: lane (arow, acol) holds column acol of rows 4 arow + r = {W1, W2 of splat 2 arow, W1, W2 of splat 2 arow + 1};
    // meaningful are W1 rows x columns 0-3 and W2 rows x columns 4-9
    const bool own1 = acol < 4;
    // writer side: where pixel lane p puts row m is wt[wbase[m / 4] + 16 m]; reader side: chunk q of this lane's row
    int wbase[4], rbase[4];
#pragma unroll
    for (int y = 0; y < 4; y++) {
        wbase[y] = GSR_WT_REGION * (lane & 3) + 4 * ((lane >> 4) ^ y) + ((lane >> 2) & 3);
        rbase[y] = GSR_WT_REGION * arow + 16 * acol + 4 * (y ^ (acol >> 2));
    }

    GSR_T_TICK(0)
    int nbatch = 0;
    for (int base = 0, taken = 0; base < total - (int)lo_pos; base += taken) {
        __syncthreads();
        GSR_T_TICK(1)
        GSR_T_COUNT(10, 1)
        nbatch++;
        const int n = min(GSR_BWD_STAGE, total - (int)lo_pos - base);
        // (round 5: one vector load per staged entry pulls its record towards this CU before the walk's scalar loads ask for it one
        // entry ahead.  With the SIMD's other waves to hide it the record's trip from HBM / the other XCDs' L2 never showed; at the end of a
        // launch, and in a launch's second round of blocks, a wave is alone with it -- 4-5 k cycles per group of eight, timing build.
        // S-room-640 K7 200 -> 170 us, walls 148 -> 142, S-1M-640 55.9 -> 55.5.)
        float touch0 = 0.f, touch1 = 0.f;
        if (tid < n) {
            const uint32_t e = point_list[range.x + (total - 1 - base - tid)];
            if (pack_qm) {          // the forward left this tile's quadrant mask of the splat in the entry (k_render_fwd, pack_qm)
                s.ids[tid] = e & 0x0FFFFFFFu;
                s.qm[tid] = (uint8_t)(e >> 28);
                const float* rr = rec + (size_t)(e & 0x0FFFFFFFu) * GSR_REC_STRIDE;
                touch0 = rr[0]; touch1 = rr[11];
            } else {
                const SplatRec sr = load_splat_rec(rec, e);
                s.ids[tid] = e;
                s.qm[tid] = (uint8_t)quadrant_mask(sr.x, sr.y, sr.a, sr.b, sr.c, sr.opacity, tx * GSR_TILE, ty * GSR_TILE);
            }
        }
        __syncthreads();
        GSR_T_TICK(2)
        // this wave's list (staged order), at most GSR_BWD_LIST entries; lim = the staged slot of the first splat that did not fit
        int cnt = 0, lim = n;
        for (int c0 = 0; c0 < n; c0 += 64) {
            const int jj = c0 + lane;
            const bool hit = jj < n && ((s.qm[min(jj, GSR_BWD_STAGE - 1)] >> wv) & 1u) && (total - base - jj) <= wave_max;
            const unsigned long long mk = __ballot(hit);
            const int at = cnt + (int)__popcll(mk & ((1ull << lane) - 1ull));
            if (hit && at < GSR_BWD_LIST) {
                s.list[wv][at] = (uint8_t)jj;
                s.off[wv][at] = s.ids[jj] * GSR_REC_STRIDE;
                s.inv[wv][jj] = (uint8_t)at;
            }
            const unsigned long long over = __ballot(hit && at == GSR_BWD_LIST);
            if (over != 0ull && lim == n) lim = c0 + (int)__builtin_ctzll(over);
            cnt = min(GSR_BWD_LIST, cnt + (int)__popcll(mk));
        }
        if (lane == 0) s.lim[wv] = lim;
        __syncthreads();
        taken = min(min(s.lim[0], s.lim[1]), min(s.lim[2], s.lim[3]));      // (>= 64 unless the tile's list ends first: a full list has 64 hits)
        // what lies beyond the end of the batch stays for the next one (the list is in staged order)
        cnt = (int)__popcll(__ballot(lane < cnt && (int)s.list[wv][min(lane, GSR_BWD_LIST - 1)] < taken));
        if (lane < ((8 - (cnt & 7)) & 7)) {      // pad to a multiple of eight with the null splat
            s.list[wv][cnt + lane] = (uint8_t)0;
            s.off[wv][cnt + lane] = (uint32_t)P * GSR_REC_STRIDE;
        }
        walked += (cnt + 7) >> 3;
        asm volatile("" : : "v"(touch0), "v"(touch1));      // (the touches have arrived: the wait sits behind the list compaction)
        GSR_T_TICK(3)
        GSR_T_COUNT(11, cnt)
        for (int g0 = 0; g0 < cnt; g0 += 8) {
            // the 8 list entries of this group in one 8-byte LDS read -> scalar registers, so that the splat
            // records of the whole group can be fetched without waiting for each other
            const unsigned long long packed = *reinterpret_cast<const unsigned long long*>(&s.list[wv][g0]);
            const uint32_t plo = __builtin_amdgcn_readfirstlane((uint32_t)packed);
            const uint32_t phi = __builtin_amdgcn_readfirstlane((uint32_t)(packed >> 32));
            const uint4 o03 = *reinterpret_cast<const uint4*>(&s.off[wv][g0]), o47 = *reinterpret_cast<const uint4*>(&s.off[wv][g0 + 4]);
#define GSR_RFL(v) ((uint32_t)__builtin_amdgcn_readfirstlane((int)(v)))
            const uint32_t offs[8] = {GSR_RFL(o03.x), GSR_RFL(o03.y), GSR_RFL(o03.z), GSR_RFL(o03.w), GSR_RFL(o47.x), GSR_RFL(o47.y), GSR_RFL(o47.z), GSR_RFL(o47.w)};
#undef GSR_RFL
            // (SIMPLE: no gradient arrives through the opacity image and the background term vanishes for every pixel of the
            // wave -- the tracking loss over a black background, i.e. the native loop: four vector instructions less per entry)
            auto bodies = [&](auto simple_tag) {
            constexpr bool SIMPLE = decltype(simple_tag)::value;
            // The entry's record: x y B2 C2 A2 opacity depth - | r g b -, wave-uniform address: scalar loads.  Scalar loads return
            // out of order, so the only wait there is for them is "all of them": the NEXT entry's record is requested right
            // after this entry's first use of its own (nothing else in flight at that point) and has the rest of the body to arrive.
            gsr_sf8 n8 = *reinterpret_cast<const GSR_CONST_AS gsr_sf8*>(crec + offs[0]);
            gsr_sf4 n4 = *reinterpret_cast<const GSR_CONST_AS gsr_sf4*>(crec + offs[0] + 8);
#pragma unroll
            for (int sidx = 0; sidx < 8; sidx++) {
                float w1 = 0.f, w2 = 0.f;
                {
                    const int j = (int)(((sidx < 4 ? plo : phi) >> (8 * (sidx & 3))) & 0xFFu);
                    const int contributor = total - base - j;
                    const gsr_sf8 r8 = n8;
                    const gsr_sf4 r4 = n4;
                    const gsr_f32x2 d = (gsr_f32x2){r8[0], r8[1]} - pxy;                  // as K6, bit for bit
                    __builtin_amdgcn_sched_barrier(0);
                    if (sidx < 7) {
                        n8 = *reinterpret_cast<const GSR_CONST_AS gsr_sf8*>(crec + offs[sidx + 1]);
                        n4 = *reinterpret_cast<const GSR_CONST_AS gsr_sf4*>(crec + offs[sidx + 1] + 8);
                    }
                    __builtin_amdgcn_sched_barrier(0);
                    const gsr_f32x2 tu = (gsr_f32x2){r8[2], r8[3]} * (gsr_f32x2){d.y, d.y};
                    const float p2 = __builtin_fmaf(d.x, __builtin_fmaf(r8[4], d.x, tu.x), tu.y * d.y);
                    const float G = __builtin_amdgcn_exp2f(p2);
                    const float alpha = fminf(0.99f, r8[5] * G);
                    const bool valid = (contributor <= last_contributor) && !(alpha < 1.0f / 255.0f) && !(p2 > 0.0f);
                    const float ae = valid ? alpha : 0.f;          // skipped => transparent: every update below is the identity
                    const float om = 1.f - ae;
                    const float r1ma = __builtin_amdgcn_rcpf(om);
                    T = T * r1ma;
                    w1 = ae * T;
                    // backward.cu:520-547 keeps four "composited behind me" recurrences (r, g, b, depth) plus the
                    // accumulated alpha, each of the form  X <- la * lastvalue + (1 - la) * X,  and then sums
                    // (value - X) * dL/dchannel.  All of it is linear in the per-splat value, so ONE recurrence on
                    //     v = c . dL/dpix + depth * dL/ddepth - dL/dalpha
                    // carries the same information:  sum_ch (value_ch - X_ch) dL_ch - (alpha - A) dL/dalpha
                    //                              = (v - V) + (1 - alpha) dL/dalpha
                    const float vc = __builtin_fmaf(r8[6], dLd, __builtin_fmaf(r4[2], dpz, __builtin_fmaf(r4[1], dpy, r4[0] * dpx)));
                    const float v = SIMPLE ? vc : vc - dLa;
                    av = __builtin_fmaf(last_alpha, lv, om_last * av);
                    float dL_dopa;
                    if (SIMPLE) dL_dopa = (v - av) * T;
                    else dL_dopa = __builtin_fmaf(__builtin_fmaf(om, dLa, v - av), T, nTf_bg * r1ma);
                    w2 = valid ? G * dL_dopa : 0.f;
                    lv = v; last_alpha = ae; om_last = om;
                }
                wt[wbase[sidx >> 1] + 16 * (2 * sidx)] = w1;
                wt[wbase[sidx >> 1] + 16 * (2 * sidx + 1)] = w2;
            }
            };
            if (simple) bodies(BoolTag<true>{}); else bodies(BoolTag<false>{});
            GSR_T_TICK(4)
            // S[16 rows = {W1,W2} x 8 splats][16 cols] += W[rows][4 pixels] * g[4 pixels][cols], 16 steps
            // (two accumulators: the 16x16x4 f32 MFMA issues every 32 cycles but a dependent one waits 40)
            gsr_f32x4 D = {0.f, 0.f, 0.f, 0.f}, D2 = {0.f, 0.f, 0.f, 0.f};
            gsr_f32x4 aop[4];
#pragma unroll
            for (int q = 0; q < 4; q++) aop[q] = *reinterpret_cast<const gsr_f32x4*>(&wt[rbase[q]]);
#pragma unroll
            for (int t = 0; t < 16; t += 2) {
                D = __builtin_amdgcn_mfma_f32_16x16x4f32(aop[t >> 2][t & 3], Breg[t], D, 0, 0, 0);
                D2 = __builtin_amdgcn_mfma_f32_16x16x4f32(aop[t >> 2][(t & 3) + 1], Breg[t + 1], D2, 0, 0, 0);
            }
            D = D + D2;
            // This wave's sums of the group's eight splats -> its slice (plain stores; padding goes to the null slot).
            if (acol < 10) {      // rows of list positions g0 + 2 arow, g0 + 2 arow + 1
                s.acc[wv][g0 + 2 * arow][acol] = own1 ? D[0] : D[1];
                s.acc[wv][g0 + 2 * arow + 1][acol] = own1 ? D[2] : D[3];
            }
            GSR_T_TICK(5)
        }
        GSR_T_TICK(6)
        __syncthreads();
        GSR_T_TICK(7)
        // per staged splat of the batch: add the slices of the waves that had it on their list (the compaction's own test),
        // recombine the moments into the nine (ten) gradient sums ...
        float* out = &s.wt[0][0];              // (the transposition buffers are idle between the walks: 4 x 1088 floats)
        if (tid < taken) {
            const uint32_t id = s.ids[tid], qmask = s.qm[tid];
            const SplatRec sr = load_splat_rec(rec, id);
            float m[10] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int w = 0; w < 4; w++)
                if (((qmask >> w) & 1u) && (total - base - tid) <= s.wmax[w]) {
                    const float* row = s.acc[w][s.inv[w][tid]];
#pragma unroll
                    for (int c = 0; c < 10; c++) m[c] += row[c];
                }
            const float M0 = m[4], Mu = m[5], Mv = m[6], Muu = m[7], Muv = m[8], Mvv = m[9];
            const float mu = sr.x - cx0, mv = sr.y - cy0, ca = sr.a, cb = sr.b, cc = sr.c, o = sr.opacity;
            const float sdx = mu * M0 - Mu, sdy = mv * M0 - Mv;
            const float sxx = mu * mu * M0 - 2.f * mu * Mu + Muu;
            const float sxy = mu * mv * M0 - mu * Mv - mv * Mu + Muv;
            const float syy = mv * mv * M0 - 2.f * mv * Mv + Mvv;
            float* q = out + tid * 10;
            q[0] = m[0]; q[1] = m[1]; q[2] = m[2];
            q[3] = -o * ddelx_dx * (ca * sdx + cb * sdy);
            q[4] = -o * ddely_dy * (cc * sdy + cb * sdx);
            q[5] = -0.5f * o * sxx;
            q[6] = -0.5f * o * sxy;
            q[7] = -0.5f * o * syy;
            q[8] = M0;
            q[9] = m[3];
            const bool nzc = q[0] != 0.f || q[1] != 0.f || q[2] != 0.f;
            const bool nz = nzc || q[3] != 0.f || q[4] != 0.f || q[5] != 0.f || q[6] != 0.f || q[7] != 0.f || q[8] != 0.f || (POSE && q[9] != 0.f);
            if (nz) aflag[id] = (uint8_t)1;
            if (nzc) aflag[(size_t)P + id] = (uint8_t)1;
        }
        __syncthreads();
        // ... and flush them: one lane per (splat, quantity), so that a wave instruction adds runs of consecutive
        // floats of the packed per-Gaussian records instead of 64 scattered rows
        for (int e = tid; e < taken * 10; e += GSR_BLOCK) {
            const int j = e / 10, q = e - j * 10;
            const float val = out[e];
            if (val != 0.f && (POSE || q != 9)) {
                // (deterministic option: the record is GSR_ACC_STRIDE pairs of 64-bit fixed-point words, see gsr_device.h)
                if (det) {
                    long long hi, lo;
                    fixed_split(val, hi, lo);
                    unsigned long long* w = reinterpret_cast<unsigned long long*>(acc) + ((size_t)s.ids[j] * GSR_ACC_STRIDE + q) * 2;
                    // (an integer cannot carry a NaN or an infinity: pair 10 of the record counts the non-finite addends, and a
                    // Gaussian that received one gets NaN gradients, as it would from the float atomics)
                    if (!__builtin_isfinite(val)) atomicAdd(reinterpret_cast<unsigned long long*>(acc) + ((size_t)s.ids[j] * GSR_ACC_STRIDE + 10) * 2, 1ull);
                    else {
                        if (hi != 0) atomicAdd(w, (unsigned long long)hi);
                        if (lo != 0) atomicAdd(w + 1, (unsigned long long)lo);
                    }
                } else atomicAdd(&acc[(size_t)s.ids[j] * GSR_ACC_STRIDE + q], val);
            }
        }
        GSR_T_TICK(8)
    }
    if (tile_work != nullptr && nseg == 1u) {      // this tile's weight in the next iteration's launch order: its longest wave + a share for the staging
        if (lane == 0) s.wmax[wv] = walked;
        __syncthreads();
        if (tid == 0) tile_work[tile] = (uint32_t)(max(max(s.wmax[0], s.wmax[1]), max(s.wmax[2], s.wmax[3])) + 2 * nbatch);
    }
    GSR_T_FLUSH(16)
}

// ---------------------------------------------------------------------------------------------
// Pose-refinement epilogue, pose state and optimiser step.
// ---------------------------------------------------------------------------------------------
// Device-resident state of one query frame's refinement (floats):
//   [0..8] R (row-major W2C rotation)  [9..11] T   [12..14] cam_rot_delta  [15..17] cam_trans_delta
//   [18] exposure_a  [19] exposure_b   [20..27] Adam exp_avg   [28..35] Adam exp_avg_sq   [36] Adam step
//   [37] converged (0/1)  [38] last loss  [39] |tau|   [48..63] viewmatrix  [64..79] projmatrix  [80..82] campos
#define GSR_PS_R 0
#define GSR_PS_T 9
#define GSR_PS_PARAM 12
#define GSR_PS_M 20
#define GSR_PS_V 28
#define GSR_PS_STEP 36
#define GSR_PS_CONV 37
#define GSR_PS_LOSS 38
#define GSR_PS_TAUN 39
#define GSR_PS_POISON 40      // uint32 bits: set by the compositing kernel when a speculative forward fails (gsr_refine)
#define GSR_PS_TICKET 41      // uint32: workgroups of the fused chain-rule kernel that have finished (native loop; returns to 0)
#define GSR_PS_BETA 84        // two doubles (floats 84-87): beta1^step, beta2^step of Adam's bias corrections
#define GSR_PS_VIEW 48
#define GSR_PS_PROJ 64
#define GSR_PS_CAMPOS 80
#define GSR_PS_PREV 96        // [96..104] R, [105..107] T, [108..109] exposure a, b as they were BEFORE the most recent pose step: the pose of the
                              // last forward / backward that ran (round 5: lets a test hold the loop's maintained gradients against the CPU restatement of the reference at that pose)
#define GSR_PS_SIZE 112

// view / proj / campos from (R, T): world_view_transform, full_proj_transform, camera_center of
// gs_localization/pipelines/tools/camera_utils.py:144-158 without the two 4x4 inversions.  Everything is read into
// registers first and written out at the end: one lane works here, and a chain of dependent LDS / global round trips (one
// per element) is what the earlier versions of the pose step spent their time on.
__device__ __forceinline__ void pose_write_camera(float* st, const float* R, const float* T, const float* proj_raw)
{
    float P[16], view[16];
#pragma unroll
    for (int i = 0; i < 16; i++) P[i] = proj_raw[i];
#pragma unroll
    for (int c = 0; c < 3; c++) {
#pragma unroll
        for (int r = 0; r < 3; r++) view[c * 4 + r] = R[r * 3 + c];
        view[c * 4 + 3] = 0.f;
    }
    view[12] = T[0]; view[13] = T[1]; view[14] = T[2]; view[15] = 1.f;
#pragma unroll
    for (int i = 0; i < 16; i++) st[GSR_PS_VIEW + i] = view[i];
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) {
            float acc = 0.f;
#pragma unroll
            for (int k = 0; k < 4; k++) acc += view[i * 4 + k] * P[k * 4 + j];
            st[GSR_PS_PROJ + i * 4 + j] = acc;
        }
#pragma unroll
    for (int c = 0; c < 3; c++) st[GSR_PS_CAMPOS + c] = -(R[0 * 3 + c] * T[0] + R[1 * 3 + c] * T[1] + R[2 * 3 + c] * T[2]);
}

__global__ void k_pose_init(float* st, const float* proj_raw)
{
    if (threadIdx.x == 0 && blockIdx.x == 0) {
        float R[9], T[3];
        for (int i = 0; i < 9; i++) R[i] = st[GSR_PS_R + i];
        for (int i = 0; i < 3; i++) T[i] = st[GSR_PS_T + i];
        pose_write_camera(st, R, T, proj_raw);
    }
}

// Every small array a gsr_refine call wants cleared before its first iteration (flags, cursors, counters, partial sums, bounds
// buffers -- a hundred KB in all), in ONE launch instead of a dozen memsets: what a 20-iteration call spends on enqueueing those
// is a fifth of an iteration each.  Ranges of 32-bit words; unused ranges have n = 0.
struct ClearRanges { uint32_t* p[14]; uint32_t n[14]; };
// gsr_refine_args.init_*: the whole initial pose state from the caller's device tensors (zeros, R, T, exposure, camera); st == nullptr: none.
// (host_state, nullable: the host's mirror of the pose state in pinned memory, see PoseStepArgs::host_state)
struct PoseLoadArgs { float* st; const float* R0; const float* T0; const float* ea; const float* eb; const float* proj_raw; float* host_state; };
__device__ __forceinline__ void pose_load_block(const PoseLoadArgs& q)          // all threads of the workgroup must call
{
    __shared__ float s_st[GSR_PS_SIZE];
    const int tid = threadIdx.x;
    for (int i = tid; i < GSR_PS_SIZE; i += blockDim.x) s_st[i] = 0.f;
    __syncthreads();
    if (tid == 0) {
        float R[9], T[3];
        for (int i = 0; i < 9; i++) R[i] = q.R0[i];
        for (int i = 0; i < 3; i++) T[i] = q.T0[i];
        for (int i = 0; i < 9; i++) s_st[GSR_PS_R + i] = R[i];
        for (int i = 0; i < 3; i++) s_st[GSR_PS_T + i] = T[i];
        s_st[GSR_PS_PARAM + 6] = q.ea[0]; s_st[GSR_PS_PARAM + 7] = q.eb[0];
        pose_write_camera(s_st, R, T, q.proj_raw);
    }
    __syncthreads();
    for (int i = tid; i < GSR_PS_SIZE; i += blockDim.x) {
        q.st[i] = s_st[i];
        if (q.host_state != nullptr) q.host_state[i] = s_st[i];
    }
}
// (the LAST workgroup loads the pose state when one is given -- one launch less in front of a call's first iteration; words of the
// state that are also listed in the ranges are zero either way)
__global__ void __launch_bounds__(GSR_BLOCK) k_refine_init(ClearRanges c, PoseLoadArgs q)
{
    if (q.st != nullptr && blockIdx.x == gridDim.x - 1) { pose_load_block(q); return; }
    const uint32_t nb = gridDim.x - (q.st != nullptr ? 1u : 0u);
    const uint32_t i0 = blockIdx.x * GSR_BLOCK + threadIdx.x, step = nb * GSR_BLOCK;
#pragma unroll
    for (int r = 0; r < 14; r++)
        for (uint32_t i = i0; i < c.n[r]; i += step) c.p[r][i] = 0u;
}

// Adam (torch.optim.Adam defaults, one lr for the four groups of 7scenes_localize_full_dslam.py:33-64) on
// [rot(3), trans(3), exposure_a, exposure_b], then update_pose (tools/pose_utils.py:54-122):
// T_w2c <- SE3_exp([trans, rot]) T_w2c, deltas <- 0, converged = |tau| < threshold.
//
// The whole pose step on one wave of 64 lanes (k_pose_step, and in the native loop the last workgroup of the chain-rule kernel,
// where it is a serial tail behind the slowest workgroup of every iteration: round 2 spent 21 k cycles here -- half of that
// kernel's duration -- in four dependent global round trips, a one-lane chain of ~1 500 instructions and a system-scope fence).
//   * every global read of the step is issued first (state, the 64 fp64 partial sums of dL/dtau, loss shards, projection):
//     one round trip; fp64 wave reductions; everything meets in LDS;
//   * Adam runs on eight lanes, one parameter each (its two correctly rounded divisions and the square root are most of the
//     one-lane chain); beta^step as running products in double (torch evaluates beta ** step in double too);
//   * SE3_exp and the camera rebuild (pose_write_camera) stay on lane 0 -- short once the rest is gone;
//   * the host gets ONE 32-bit status word (native loop): (seq << 4) | overflow << 2 | bound failure << 1 | converged -- a single
//     store needs no fence; loss and |tau| stay in the state, which the host copies out once at the end of the call.
// tau_acc (nullable): the fp64 block sums of K8/K9; when given, the step also finishes the dL/dtau reduction (writes
// dL_dtau_out).  loss_shards (nullable): the native loop's fused-loss partial sums.  Whether or not the update runs (a failed
// or frozen group only publishes its status), the loss shards and the superblock bounds the next forward accumulates into
// (clear_b) are cleared here: the last workgroup of every group does it, so a failed forward leaves nothing behind.
#define GSR_TAU_SLOTS 64      // partial sums of dL/dtau (k_preprocess_bwd), 64 B apart
// dL/dtau from the twelve world-frame sums of the chain-rule kernel (k_preprocess_bwd, (6)): sw[0..2] the rho part, [3..5] sum g_geo,
// [6..8] sum p x g_geo, [9..11] sum 2 a; Wc[r][c] = vm[4 c + r], trans = vm[12..14].
__device__ __forceinline__ void tau_from_world_sums(const double* sw, const float* vm, double* tau)
{
    double wg[3];
#pragma unroll
    for (int r = 0; r < 3; r++) {
        const double w0 = vm[r], w1 = vm[4 + r], w2 = vm[8 + r];          // row r of Wc
        tau[r] = w0 * sw[0] + w1 * sw[1] + w2 * sw[2];
        wg[r] = w0 * sw[3] + w1 * sw[4] + w2 * sw[5];
        tau[3 + r] = w0 * (sw[6] + sw[9]) + w1 * (sw[7] + sw[10]) + w2 * (sw[8] + sw[11]);
    }
    const double t0 = vm[12], t1 = vm[13], t2 = vm[14];
    tau[3] += t1 * wg[2] - t2 * wg[1]; tau[4] += t2 * wg[0] - t0 * wg[2]; tau[5] += t0 * wg[1] - t1 * wg[0];
}
struct PoseStepArgs {
    float* st; const float* dL_dtau; double* tau_acc; float* dL_dtau_out; const float* loss_out; const float* proj_raw;
    float lr, conv_thr; float* loss_zero; uint32_t* host_status; int seq; float* loss_shards; float* clear_b; int clear_n;
    int det;        // deterministic option: tau_acc holds 12 fixed-point world-frame sums per slot, loss_shards fixed-point sums
    float* host_state;      // nullable, pinned host memory, GSR_PS_SIZE floats: every step that runs mirrors the new state there, so that the
                            // call can hand the final pose back without a device-to-host copy in front of its last synchronisation
    float* prev_cam;        // nullable, 35 floats: view (16), projection (16), camera position (3) as they were BEFORE this step -- the camera of
                            // the iteration whose records the final pass of k_preprocess_bwd turns into gradient rows (PreBwdArgs::role)
};
struct alignas(16) PoseStepLDS { float st[GSR_PS_SIZE]; float t6[8]; float loss[4]; float proj[16]; };
template <bool DET>      // (compile time: the deterministic option's branches cost the default path's serial tail 2 k cycles as run-time tests)
__device__ __forceinline__ void pose_step_wave(const PoseStepArgs& q, LoopGuard guard, PoseStepLDS& s)
{
    const bool run = !guard.frozen();          // wave-uniform
    const int lane = threadIdx.x & 63;
    float* st = q.st;
    const uint32_t pz = guard.poison ? *guard.poison : 0u;
    // (1) every global read first
    float va = 0.f, vb = 0.f, ls = 0.f, pj = 0.f, tq = 0.f;
    double tv[6] = {0.0, 0.0, 0.0, 0.0, 0.0, 0.0};
    long long tvi[12] = {0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0}, tvn = 0, lsi = 0;
    constexpr bool det = DET;
    if (run) {
        va = st[lane];
        if (lane < GSR_PS_SIZE - 64) vb = st[64 + lane];
        if (q.tau_acc != nullptr && det) {     // (deterministic option: the twelve world-frame sums of tau_pack, fixed point; second half behind the slots)
            const long long* ta = reinterpret_cast<const long long*>(q.tau_acc);
#pragma unroll
            for (int i = 0; i < 12; i++)
                tvi[i] = __hip_atomic_load(&ta[(i < 6 ? 0 : 8 * GSR_TAU_SLOTS) + lane * 8 + (i < 6 ? i : i - 6)], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            tvn = __hip_atomic_load(&ta[lane * 8 + 7], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);      // (Gaussians whose terms were not finite)
        } else if (q.tau_acc != nullptr) {     // lane = slot: 64 partial sums per component (other workgroups of this launch added to them:
#pragma unroll                                 //  agent-scope atomic loads, past this CU's L1)
            for (int i = 0; i < 6; i++) tv[i] = __hip_atomic_load(&q.tau_acc[lane * 8 + i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        } else if (lane < 6) tq = q.dL_dtau[lane];
        if (lane < 16) pj = q.proj_raw[lane];
    }
    // fused loss: lane = shard * 4 + component
    if (q.loss_shards != nullptr && det) {
        long long* sh = reinterpret_cast<long long*>(q.loss_shards + (lane >> 2) * 16) + (lane & 3);      // (component 3: unused, zero)
        if (run) lsi = *sh;
        *sh = 0;
    } else if (q.loss_shards != nullptr) {
        const int at = (lane >> 2) * 16 + (lane & 3);
        if (run) ls = q.loss_shards[at];
        q.loss_shards[at] = 0.f;               // (also what a failed forward added)
    } else if (run && lane < 4) ls = q.loss_out[lane];
    if (q.clear_b != nullptr)                  // per-superblock bounds the next forward accumulates into
        for (int i = lane; i < q.clear_n; i += 64) q.clear_b[i] = 0.f;
    float conv_out = 0.f;
    if (run) {
        s.st[lane] = va;
        if (lane < GSR_PS_SIZE - 64) s.st[64 + lane] = vb;
        // (the pose and exposure this group's forward and backward ran with: GSR_PS_PREV; a wave executes in order, no barrier needed)
        if (lane < 12) s.st[GSR_PS_PREV + lane] = va;
        if (lane == GSR_PS_PARAM + 6 || lane == GSR_PS_PARAM + 7) s.st[GSR_PS_PREV + 12 + lane - (GSR_PS_PARAM + 6)] = va;
        if (q.prev_cam != nullptr) {
            static_assert(GSR_PS_VIEW == 48 && GSR_PS_PROJ == 64 && GSR_PS_CAMPOS == 80, "prev_cam is copied by lane from these places");
            if (lane >= GSR_PS_VIEW) q.prev_cam[lane - GSR_PS_VIEW] = va;
            if (lane < 19) q.prev_cam[16 + lane] = vb;
        }
        if (q.tau_acc != nullptr && det) {
            double sw[12];
#pragma unroll
            for (int i = 0; i < 12; i++) sw[i] = from_fixed(wave_sum_ll_to_lane63(tvi[i]), GSR_FIX_TAU);
            // the view matrix of this iteration sits in lanes 48 ... 63 of `va` (state words GSR_PS_VIEW ...)
            float vmx[16];
#pragma unroll
            for (int k = 0; k < 16; k++) vmx[k] = __uint_as_float((uint32_t)__builtin_amdgcn_readlane((int)__float_as_uint(va), GSR_PS_VIEW + k));
            const long long nonfinite = wave_sum_ll_to_lane63(tvn);
            if (lane == 63) {
                double tau[6];
                tau_from_world_sums(sw, vmx, tau);
#pragma unroll
                for (int i = 0; i < 6; i++) s.t6[i] = (nonfinite != 0) ? __builtin_nanf("") : (float)tau[i];
            }
            if (q.loss_zero != nullptr) {
                long long* ta = reinterpret_cast<long long*>(q.tau_acc);
#pragma unroll
                for (int i = 0; i < 6; i++) { ta[lane * 8 + i] = 0; ta[8 * GSR_TAU_SLOTS + lane * 8 + i] = 0; }
                ta[lane * 8 + 7] = 0;
            }
        } else if (q.tau_acc != nullptr) {
#pragma unroll
            for (int i = 0; i < 6; i++) {
                const double t = wave_sum_d_to_lane63(tv[i]);
                if (lane == 63) s.t6[i] = (float)t;
            }
            if (q.loss_zero != nullptr) {      // native loop: leave the partial sums clean for the next backward
#pragma unroll
                for (int i = 0; i < 6; i++) q.tau_acc[lane * 8 + i] = 0.0;
            }
        } else if (lane < 6) s.t6[lane] = tq;
        if (q.loss_shards != nullptr && det) {
#pragma unroll
            for (int off = 4; off < 64; off <<= 1) lsi += __shfl_xor(lsi, off, 64);
            ls = (__shfl(lsi, 3, 64) != 0) ? __builtin_nanf("") : (float)from_fixed(lsi, GSR_FIX_LOSS);      // (component 3: non-finite tile sums seen)
        } else if (q.loss_shards != nullptr) {
#pragma unroll
            for (int off = 4; off < 64; off <<= 1) ls += __shfl_xor(ls, off, 64);
        }
        if (lane < 4) s.loss[lane] = ls;
        if (lane < 16) s.proj[lane] = pj;
        __syncthreads();
        // (2) Adam, one parameter per lane: [rot(3), trans(3), exposure_a, exposure_b] <- gradients [theta(3), rho(3), da, db]
        const float step = s.st[GSR_PS_STEP] + 1.f;
        const double* beta = reinterpret_cast<const double*>(s.st + GSR_PS_BETA);
        const double b1t = (step == 1.f ? 1.0 : beta[0]) * 0.9, b2t = (step == 1.f ? 1.0 : beta[1]) * 0.999;
        const double bc1 = 1.0 - b1t, bc2 = 1.0 - b2t;
        const float step_size = (float)((double)q.lr / bc1);
        const float bc2_sqrt = (float)sqrt(bc2);
        const float w1 = (float)(1.0 - 0.9), w2 = (float)(1.0 - 0.999);
        float par = 0.f, m = 0.f, v = 0.f;
        if (lane < 8) {
            const float g = (lane < 3) ? s.t6[3 + lane] : ((lane < 6) ? s.t6[lane - 3] : s.loss[lane - 5]);
            m = s.st[GSR_PS_M + lane]; v = s.st[GSR_PS_V + lane]; par = s.st[GSR_PS_PARAM + lane];
            m = m + w1 * (g - m);                                  // exp_avg.lerp_(grad, 1 - beta1)
            v = v * 0.999f + w2 * (g * g);                         // exp_avg_sq.mul_(beta2).addcmul_(grad, grad, 1 - beta2)
            const float denom = sqrtf(v) / bc2_sqrt + 1e-8f;
            par = par + (-step_size) * (m / denom);
        }
        __syncthreads();                       // (everybody has read the old state)
        if (lane < 8) { s.st[GSR_PS_M + lane] = m; s.st[GSR_PS_V + lane] = v; }
        if (lane == 6 || lane == 7) s.st[GSR_PS_PARAM + lane] = par;
        if (lane < 6) {
            s.st[GSR_PS_PARAM + lane] = 0.f;                       // cam_rot_delta / cam_trans_delta .fill_(0)
            if (q.tau_acc != nullptr && q.dL_dtau_out != nullptr) q.dL_dtau_out[lane] = s.t6[lane];
        }
#define GSR_RL(k) __uint_as_float((uint32_t)__builtin_amdgcn_readlane((int)__float_as_uint(par), k))
        const float th[3] = {GSR_RL(0), GSR_RL(1), GSR_RL(2)}, rho[3] = {GSR_RL(3), GSR_RL(4), GSR_RL(5)};
#undef GSR_RL
        // (3) update_pose on lane 0
        if (lane == 0) {
            float R[9], T[3];
#pragma unroll
            for (int i = 0; i < 9; i++) R[i] = s.st[GSR_PS_R + i];
#pragma unroll
            for (int i = 0; i < 3; i++) T[i] = s.st[GSR_PS_T + i];
            const float Wm[9] = {0.f, -th[2], th[1], th[2], 0.f, -th[0], -th[1], th[0], 0.f};
            float W2[9];
#pragma unroll
            for (int i = 0; i < 3; i++)
#pragma unroll
                for (int j = 0; j < 3; j++) W2[i * 3 + j] = Wm[i * 3] * Wm[j] + Wm[i * 3 + 1] * Wm[3 + j] + Wm[i * 3 + 2] * Wm[6 + j];
            const float angle = sqrtf(th[0] * th[0] + th[1] * th[1] + th[2] * th[2]);
            float cW, cW2, vW, vW2;
            if (angle < 1e-5f) { cW = 1.f; cW2 = 0.5f; vW = 0.5f; vW2 = 1.0f / 6.0f; }
            else {
                cW = sinf(angle) / angle; cW2 = (1.f - cosf(angle)) / (angle * angle);
                vW = (1.0f - cosf(angle)) / (angle * angle); vW2 = (angle - sinf(angle)) / (angle * angle * angle);
            }
            float Re[9], Vm[9];
#pragma unroll
            for (int i = 0; i < 9; i++) {
                const float I = (i == 0 || i == 4 || i == 8) ? 1.f : 0.f;
                Re[i] = I + cW * Wm[i] + cW2 * W2[i];
                Vm[i] = I + Wm[i] * vW + W2[i] * vW2;
            }
            float te[3], Rn[9], Tn[3];
#pragma unroll
            for (int i = 0; i < 3; i++) te[i] = Vm[i * 3] * rho[0] + Vm[i * 3 + 1] * rho[1] + Vm[i * 3 + 2] * rho[2];
#pragma unroll
            for (int i = 0; i < 3; i++) {
#pragma unroll
                for (int j = 0; j < 3; j++) Rn[i * 3 + j] = Re[i * 3] * R[j] + Re[i * 3 + 1] * R[3 + j] + Re[i * 3 + 2] * R[6 + j];
                Tn[i] = Re[i * 3] * T[0] + Re[i * 3 + 1] * T[1] + Re[i * 3 + 2] * T[2] + te[i];
            }
            const float taun = sqrtf(rho[0] * rho[0] + rho[1] * rho[1] + rho[2] * rho[2] + th[0] * th[0] + th[1] * th[1] + th[2] * th[2]);
            s.st[GSR_PS_STEP] = step;
            double* beta_w = reinterpret_cast<double*>(s.st + GSR_PS_BETA);
            beta_w[0] = b1t; beta_w[1] = b2t;
#pragma unroll
            for (int i = 0; i < 9; i++) s.st[GSR_PS_R + i] = Rn[i];
#pragma unroll
            for (int i = 0; i < 3; i++) s.st[GSR_PS_T + i] = Tn[i];
            s.st[GSR_PS_CONV] = (taun < q.conv_thr) ? 1.f : 0.f;
            s.st[GSR_PS_TAUN] = taun;
            s.st[GSR_PS_LOSS] = s.loss[0];
            pose_write_camera(s.st, Rn, Tn, s.proj);
        }
        __syncthreads();
        conv_out = s.st[GSR_PS_CONV];
        for (int i = lane; i < GSR_PS_SIZE; i += 64)
            if (i != GSR_PS_POISON && i != GSR_PS_TICKET) {           // (those two words belong to other kernels and the host)
                st[i] = s.st[i];
                if (q.host_state != nullptr) q.host_state[i] = s.st[i];
            }
        if (q.loss_zero != nullptr && lane < 4) q.loss_zero[lane] = 0.f;
    } else conv_out = st[GSR_PS_CONV];
    if (lane == 0 && q.host_status != nullptr) {
        const uint32_t flags = ((pz >> 2) == guard.tag && guard.poison != nullptr) ? (pz & 3u) : 0u;
        // one 32-bit store into pinned host memory: the host polls the sequence bits and finds the flags in the same word
        *reinterpret_cast<volatile uint32_t*>(q.host_status) = ((uint32_t)q.seq << 4) | (flags << 1) | (conv_out != 0.f ? 1u : 0u);
    }
}
__global__ void __launch_bounds__(64) k_pose_step(PoseStepArgs q, LoopGuard guard)
{
    __shared__ PoseStepLDS s;
    if (blockIdx.x == 0) pose_step_wave<false>(q, guard, s);
}

// ---------------------------------------------------------------------------------------------
// K8+K9  per-Gaussian chain rule (replaces backward.cu:144-274 computeCov2DCUDA and :346-396
// preprocessCUDA, fused into one pass) + the SE(3) pose-gradient reduction of the pose package.
// One lane per Gaussian; HBM-streaming.  Every output element is written exactly once.
// ---------------------------------------------------------------------------------------------
struct PreBwdArgs {
    int P, D, M;
    const float* means; const int* radii; const float* shs; const uint8_t* clamped;
    const float* scales; const float* rots; float mod; const float* cov3D;   // cov3D: precomp or geom state
    const float* rec;                                     // the forward's packed splat records (the conic it used)
    const float* view; const float* proj; const float* campos;
    float fx, fy, tanx, tany;
    float* acc;                                           // packed K7 sums, GSR_ACC_STRIDE floats per Gaussian
    float* dL_dmean2D; float* dL_dconic; float* dL_dopacity; float* dL_dcolor;      // unpacked here, written once
    float* dL_dmean3D; float* dL_dcov3D; float* dL_dsh; float* dL_dscale; float* dL_drot;
    int pose; double* tau_acc;
    // Native loop only (nullable).  The gradient tensors are then zero-filled ONCE and kept consistent from one
    // iteration to the next: bit 0 = this Gaussian's small gradient rows hold values, bit 1 = its dL_dsh row does.
    // A row is re-zeroed only when it held values and gets none this time, instead of 300 MB of memsets per call.
    uint8_t* dirty;
    uint8_t* aflag;                                       // 2 P bytes, set by k_render_bwd_mfma: has sums / has colour sums; cleared here as consumed
    LoopGuard guard;
    SurvLists surv; // the forward's work lists (k_preprocess): the only Gaussians whose records can hold anything
    // Native loop (role != 0): the gradients of the Gaussians' own parameters are read by nobody before the call returns, so an
    // iteration's launch only computes dL/dtau (no gradient rows, no dirty bits, nothing consumed) and the rows are written ONCE, from
    // the records of the last iteration whose pose step ran.  For that the groups alternate between two sets of work lists / flags /
    // records: a group's launch walks its OWN set for dL/dtau and clears what its predecessor left in the OTHER one (o_*), whose list
    // counters its last workgroup returns to zero for the forward after next.
    //   role 1  a group's launch.  Not frozen: dL/dtau from the own set, the other set cleared.  Poisoned (this group's forward failed
    //           its verification): the other set cleared.  Converged: the group in front of this one was the last iteration -- its set
    //           (o_*) gets the full treatment, rows and dirty bits, once (*final_done), before a later frozen forward reuses its lists.
    //   role 2  launched by the host behind the last group: the full treatment of o_* unless *final_done says it has been given.
    int role;
    int rows_every;      // GSR_REFINE_GRADS_EVERY_ITERATION (diagnostics): role 1 launches write the rows themselves, no final pass
    SurvLists o_surv; uint8_t* o_aflag; float* o_acc; uint32_t* final_done;
    const float* o_rec; const uint8_t* o_clamped;      // (the splat records and SH clamp flags of that set's forward ...
    const float* o_cam;                                // ... and its camera: PoseStepArgs::prev_cam)
    // Native loop only (ticket nullable): the workgroup that finishes LAST runs the pose step (Adam, update_pose, camera
    // matrices, status for the host) right here instead of in a launch of its own: every workgroup bumps the ticket once its
    // dL/dtau sums are out; whoever draws the last number sees all of them.
    uint32_t* ticket; PoseStepArgs fold;
};

// ---- chain rule of one Gaussian, written from the maths rather than from the reference's expression trees -------------
// Notation: p world mean, t = Wc p + trans its camera-space position (Wc[r][c] = view[4 c + r]), J the 2x3 perspective
// Jacobian (backward.cu:166-199 keeps the clamped x/z, y/z in it as constants), M = J Wc (2x3), C = M Sigma M^T + 0.3 I the
// screen-space covariance and Q = C^-1 the conic.  All gradient matrices below are the SYMMETRIC ones (an off-diagonal
// parameter that appears twice gets half of its total derivative in each place).

// Colour gradient -> SH coefficient gradients and the gradient w.r.t. the mean through the view direction
// (what backward.cu:20-139 computes).  colour_c = max(0, sum_k B_k(d) sh[k][c] + 0.5), d = (p - campos) / |p - campos|:
//   dL/dsh[k][c] = B_k(d) g_c                      g = dL/dcolour with the clamped channels masked
//   dL/dd        = sum_k (sh[k] . g) grad B_k(d)   (x, y, z treated as independent, then projected through the
//   dL/dp        = (dL/dd - d (d . dL/dd)) / |p - campos|                                  normalisation)
// dsh may alias sh: row k is read before it is written.
__device__ __forceinline__ float3 sh_color_backward(int deg, int M, float3 pos, const float* campos, const float* sh, uint8_t clamp_bits,
                                                    float3 dcol, float* dsh)
{
    const float3 v = make_float3(pos.x - campos[0], pos.y - campos[1], pos.z - campos[2]);
    const float rlen = 1.0f / sqrtf(v.x * v.x + v.y * v.y + v.z * v.z);
    const float x = v.x * rlen, y = v.y * rlen, z = v.z * rlen;
    const float g0 = (clamp_bits & 1) ? 0.f : dcol.x, g1 = (clamp_bits & 2) ? 0.f : dcol.y, g2 = (clamp_bits & 4) ? 0.f : dcol.z;
    float dx = 0.f, dy = 0.f, dz = 0.f;
    // one term of the expansion: basis value b, basis gradient (bx, by, bz)
#define GSR_SH_TERM(k, b, bx, by, bz)                                                                         \
    {                                                                                                         \
        const float c_ = sh[(k) * 3] * g0 + sh[(k) * 3 + 1] * g1 + sh[(k) * 3 + 2] * g2;                      \
        dx += c_ * (bx); dy += c_ * (by); dz += c_ * (bz);                                                    \
        if (dsh) { const float b_ = (b); dsh[(k) * 3] = b_ * g0; dsh[(k) * 3 + 1] = b_ * g1; dsh[(k) * 3 + 2] = b_ * g2; } \
    }
    if (dsh) { dsh[0] = kSH_C0 * g0; dsh[1] = kSH_C0 * g1; dsh[2] = kSH_C0 * g2; }
    if (deg > 0) {
        GSR_SH_TERM(1, -kSH_C1 * y, 0.f, -kSH_C1, 0.f)
        GSR_SH_TERM(2, kSH_C1 * z, 0.f, 0.f, kSH_C1)
        GSR_SH_TERM(3, -kSH_C1 * x, -kSH_C1, 0.f, 0.f)
        if (deg > 1) {
            const float xx = x * x, yy = y * y, zz = z * z, xy = x * y, yz = y * z, xz = x * z;
            GSR_SH_TERM(4, kSH_C2[0] * xy, kSH_C2[0] * y, kSH_C2[0] * x, 0.f)
            GSR_SH_TERM(5, kSH_C2[1] * yz, 0.f, kSH_C2[1] * z, kSH_C2[1] * y)
            GSR_SH_TERM(6, kSH_C2[2] * (2.f * zz - xx - yy), kSH_C2[2] * (-2.f * x), kSH_C2[2] * (-2.f * y), kSH_C2[2] * (4.f * z))
            GSR_SH_TERM(7, kSH_C2[3] * xz, kSH_C2[3] * z, 0.f, kSH_C2[3] * x)
            GSR_SH_TERM(8, kSH_C2[4] * (xx - yy), kSH_C2[4] * (2.f * x), kSH_C2[4] * (-2.f * y), 0.f)
            if (deg > 2) {
                GSR_SH_TERM(9, kSH_C3[0] * y * (3.f * xx - yy), kSH_C3[0] * (6.f * xy), kSH_C3[0] * (3.f * xx - 3.f * yy), 0.f)
                GSR_SH_TERM(10, kSH_C3[1] * xy * z, kSH_C3[1] * yz, kSH_C3[1] * xz, kSH_C3[1] * xy)
                GSR_SH_TERM(11, kSH_C3[2] * y * (4.f * zz - xx - yy), kSH_C3[2] * (-2.f * xy), kSH_C3[2] * (4.f * zz - xx - 3.f * yy), kSH_C3[2] * (8.f * yz))
                GSR_SH_TERM(12, kSH_C3[3] * z * (2.f * zz - 3.f * xx - 3.f * yy), kSH_C3[3] * (-6.f * xz), kSH_C3[3] * (-6.f * yz),
                            kSH_C3[3] * (6.f * zz - 3.f * xx - 3.f * yy))
                GSR_SH_TERM(13, kSH_C3[4] * x * (4.f * zz - xx - yy), kSH_C3[4] * (4.f * zz - 3.f * xx - yy), kSH_C3[4] * (-2.f * xy), kSH_C3[4] * (8.f * xz))
                GSR_SH_TERM(14, kSH_C3[5] * z * (xx - yy), kSH_C3[5] * (2.f * xz), kSH_C3[5] * (-2.f * yz), kSH_C3[5] * (xx - yy))
                GSR_SH_TERM(15, kSH_C3[6] * x * (xx - 3.f * yy), kSH_C3[6] * (3.f * xx - 3.f * yy), kSH_C3[6] * (-6.f * xy), 0.f)
            }
        }
    }
#undef GSR_SH_TERM
    if (dsh)      // coefficients above the active degree receive zero gradient (the reference's buffer is pre-zeroed)
        for (int k = (deg + 1) * (deg + 1); k < M; k++) { dsh[k * 3] = 0.f; dsh[k * 3 + 1] = 0.f; dsh[k * 3 + 2] = 0.f; }
    const float along = x * dx + y * dy + z * dz;
    return make_float3((dx - x * along) * rlen, (dy - y * along) * rlen, (dz - z * along) * rlen);
}

// Screen-space gradients of one Gaussian -> gradient of its 3D covariance and of its mean through the projection of the
// covariance (what backward.cu:144-274 computes).  Inputs: the conic Q the forward stored, gq = dL/d(Qa, Qb, Qc) as the
// compositing backward sums them (Qb appears once in the exponent).
//   H  = dL/dC = -Q Gq Q,  Gq = [[gq.x, gq.y], [gq.y, gq.z]]          (derivative of the matrix inverse)
//   G3 = dL/dSigma = M^T H M                                           (6 unique entries; out_G)
//   D  = dL/dM = 2 H (M Sigma)
//   dL/dJ = D Wc^T restricted to J's four non-constant entries, then dL/dt through J(t), then dL/dp = Wc^T dL/dt.
__device__ __forceinline__ float3 covariance_chain(float3 p, const float* cov6, float3 Q, float3 gq, const float* view, float fx, float fy,
                                                   float tanx, float tany, float* out_G)
{
    const float W00 = view[0], W01 = view[4], W02 = view[8], W10 = view[1], W11 = view[5], W12 = view[9], W20 = view[2], W21 = view[6],
                W22 = view[10];
    const float tx = W00 * p.x + W01 * p.y + W02 * p.z + view[12], ty = W10 * p.x + W11 * p.y + W12 * p.z + view[13],
                tz = W20 * p.x + W21 * p.y + W22 * p.z + view[14];
    const float rz = 1.0f / tz, rz2 = rz * rz;
    const float limx = 1.3f * tanx, limy = 1.3f * tany;
    const float ux = tx * rz, uy = ty * rz;
    const bool in_x = !(ux < -limx || ux > limx), in_y = !(uy < -limy || uy > limy);
    const float cx = fminf(limx, fmaxf(-limx, ux)) * tz, cy = fminf(limy, fmaxf(-limy, uy)) * tz;      // the clamped t.x, t.y of the forward
    const float j00 = fx * rz, j02 = -fx * cx * rz2, j11 = fy * rz, j12 = -fy * cy * rz2;
    const float m0[3] = {j00 * W00 + j02 * W20, j00 * W01 + j02 * W21, j00 * W02 + j02 * W22};
    const float m1[3] = {j11 * W10 + j12 * W20, j11 * W11 + j12 * W21, j11 * W12 + j12 * W22};
    const float u00 = Q.x * gq.x + Q.y * gq.y, u01 = Q.x * gq.y + Q.y * gq.z, u10 = Q.y * gq.x + Q.z * gq.y, u11 = Q.y * gq.y + Q.z * gq.z;
    const float h00 = -(u00 * Q.x + u01 * Q.y), h01 = -(u00 * Q.y + u01 * Q.z), h11 = -(u10 * Q.y + u11 * Q.z);
    float n0[3], n1[3];
#pragma unroll
    for (int k = 0; k < 3; k++) { n0[k] = h00 * m0[k] + h01 * m1[k]; n1[k] = h01 * m0[k] + h11 * m1[k]; }
    out_G[0] = m0[0] * n0[0] + m1[0] * n1[0]; out_G[1] = m0[0] * n0[1] + m1[0] * n1[1]; out_G[2] = m0[0] * n0[2] + m1[0] * n1[2];
    out_G[3] = m0[1] * n0[1] + m1[1] * n1[1]; out_G[4] = m0[1] * n0[2] + m1[1] * n1[2]; out_G[5] = m0[2] * n0[2] + m1[2] * n1[2];
    const float S[3][3] = {{cov6[0], cov6[1], cov6[2]}, {cov6[1], cov6[3], cov6[4]}, {cov6[2], cov6[4], cov6[5]}};
    // (D = 2 H (M Sigma): the reference's order of the two products -- (H M) Sigma is the same matrix, with larger intermediate terms
    // for thin splats)
    float k0[3], k1[3];
#pragma unroll
    for (int k = 0; k < 3; k++) {
        k0[k] = m0[0] * S[0][k] + m0[1] * S[1][k] + m0[2] * S[2][k];
        k1[k] = m1[0] * S[0][k] + m1[1] * S[1][k] + m1[2] * S[2][k];
    }
    float d0[3], d1[3];
#pragma unroll
    for (int k = 0; k < 3; k++) {
        d0[k] = 2.f * (h00 * k0[k] + h01 * k1[k]);
        d1[k] = 2.f * (h01 * k0[k] + h11 * k1[k]);
    }
    const float e00 = d0[0] * W00 + d0[1] * W01 + d0[2] * W02, e02 = d0[0] * W20 + d0[1] * W21 + d0[2] * W22;
    const float e11 = d1[0] * W10 + d1[1] * W11 + d1[2] * W12, e12 = d1[0] * W20 + d1[1] * W21 + d1[2] * W22;
    const float dtx = in_x ? -fx * rz2 * e02 : 0.f, dty = in_y ? -fy * rz2 * e12 : 0.f;
    const float dtz = -rz2 * (fx * e00 + fy * e11) + 2.f * rz2 * rz * (fx * cx * e02 + fy * cy * e12);
    return make_float3(W00 * dtx + W10 * dty + W20 * dtz, W01 * dtx + W11 * dty + W21 * dtz, W02 * dtx + W12 * dty + W22 * dtz);
}

// dL/dSigma (symmetric, G = G00 G01 G02 G11 G12 G22) -> gradients of the scale and of the quaternion used AS GIVEN
// (what backward.cu:278-341 computes).  Sigma = R S^2 R^T, S = diag(mod * scale), R the rotation of q = (r, x, y, z):
//   dL/ds_j = 2 s_j (R^T G R)_jj,   dL/dR = 2 G R S^2 =: E,   dL/dq = sum_ij E_ij dR_ij/dq.
__device__ __forceinline__ void covariance_param_grads(const float* scale3, float mod, float4 q, const float* G, float* dscale, float* dq)
{
    const float r = q.x, x = q.y, y = q.z, z = q.w;
    const float R[3][3] = {{1.f - 2.f * (y * y + z * z), 2.f * (x * y - r * z), 2.f * (x * z + r * y)},
                           {2.f * (x * y + r * z), 1.f - 2.f * (x * x + z * z), 2.f * (y * z - r * x)},
                           {2.f * (x * z - r * y), 2.f * (y * z + r * x), 1.f - 2.f * (x * x + y * y)}};
    const float Gm[3][3] = {{G[0], G[1], G[2]}, {G[1], G[3], G[4]}, {G[2], G[4], G[5]}};
    float A[3][3];
#pragma unroll
    for (int i = 0; i < 3; i++)
#pragma unroll
        for (int j = 0; j < 3; j++) A[i][j] = Gm[i][0] * R[0][j] + Gm[i][1] * R[1][j] + Gm[i][2] * R[2][j];
    float E[3][3];
#pragma unroll
    for (int j = 0; j < 3; j++) {
        const float sj = mod * scale3[j];
        dscale[j] = mod * 2.f * sj * (R[0][j] * A[0][j] + R[1][j] * A[1][j] + R[2][j] * A[2][j]);
        const float w = 2.f * sj * sj;
#pragma unroll
        for (int i = 0; i < 3; i++) E[i][j] = w * A[i][j];
    }
    dq[0] = 2.f * (z * (E[1][0] - E[0][1]) + y * (E[0][2] - E[2][0]) + x * (E[2][1] - E[1][2]));
    dq[1] = 2.f * (y * (E[0][1] + E[1][0]) + z * (E[0][2] + E[2][0]) + r * (E[2][1] - E[1][2])) - 4.f * x * (E[1][1] + E[2][2]);
    dq[2] = 2.f * (x * (E[0][1] + E[1][0]) + r * (E[0][2] - E[2][0]) + z * (E[1][2] + E[2][1])) - 4.f * y * (E[0][0] + E[2][2]);
    dq[3] = 2.f * (r * (E[1][0] - E[0][1]) + x * (E[0][2] + E[2][0]) + y * (E[1][2] + E[2][1])) - 4.f * z * (E[0][0] + E[1][1]);
}

// One WAVE per 64-entry chunk of a work list (workgroup = 64 lanes, ~15 KB of LDS, no cross-wave barriers; workgroup w walks
// sub-list w mod GSR_SURV_LISTS from chunk w / GSR_SURV_LISTS in steps of gridDim / GSR_SURV_LISTS).  Every lane looks at
// one survivor's accumulator record; the ones K7 added anything to run the chain rule, SH rows staged through LDS.
// The kernel is bound by the latency of a wave's dependent phases (list -> record -> parameter gathers -> chain rule ->
// stores) at the 2 waves per SIMD its registers allow, so the host launches at most as many waves as are resident at once.
// (Round 1 / early round 2 scanned all P Gaussians' records for the active ones: 48 MB per iteration at 1 M Gaussians for the
// ~4 % that had work.)
#define GSR_K8_ROWS 64
#define GSR_K8_RESIDENT (256 * 4 * 2)
// K7's record of one Gaussian: twelve floats, or (DET, the deterministic option) twelve (coarse, fine) pairs of 64-bit fixed-point words
template <bool DET>
__device__ __forceinline__ void acc_load(const float* acc, size_t idx, float4& r0, float4& r1, float4& r2)
{
    if (DET) {
        const longlong2* w = reinterpret_cast<const longlong2*>(acc) + idx * GSR_ACC_STRIDE;      // one (hi, lo) pair per quantity
        float q[10];
#pragma unroll
        for (int i = 0; i < 10; i++) { const longlong2 p = w[i]; q[i] = (float)fixed_join(p.x, p.y); }
        if (w[10].x != 0) {          // a non-finite addend arrived (see the flush of k_render_bwd_mfma)
#pragma unroll
            for (int i = 0; i < 10; i++) q[i] = __builtin_nanf("");
        }
        r0 = make_float4(q[0], q[1], q[2], q[3]);
        r1 = make_float4(q[4], q[5], q[6], q[7]);
        r2 = make_float4(q[8], q[9], 0.f, 0.f);
    } else {
        const float4* rec = reinterpret_cast<const float4*>(acc + idx * GSR_ACC_STRIDE);
        r0 = rec[0]; r1 = rec[1]; r2 = rec[2];
    }
}
template <bool DET>
__device__ __forceinline__ void acc_clear(float* acc, size_t idx)
{
    float4* rec = DET ? reinterpret_cast<float4*>(acc) + idx * GSR_ACC_STRIDE : reinterpret_cast<float4*>(acc + idx * GSR_ACC_STRIDE);
    const float4 z = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int i = 0; i < (DET ? 11 : 3); i++) rec[i] = z;
}
// Stateless backward, one launch in front of k_render_bwd_mfma:
//   * K7's accumulator records and flags must start from zero, and only the survivors of the forward can be on a tile's list -- their
//     records are cleared by walking the work lists (1.5 M Gaussians of which a third to a half are survivors: 48 B each instead of
//     a 72 MB memset; acc == nullptr: the host cleared them).  Workgroup w: sub-list w mod GSR_SURV_LISTS, 1 024-entry chunks
//     w / GSR_SURV_LISTS, ... in steps of clear_blocks / GSR_SURV_LISTS;
//   * the FIRST workgroup computes K7's launch order from the work the forward measured (tile_order_block; order == nullptr: none).
//     On its own that is a 19 us kernel for 4 293 tiles (one workgroup, a chain of dependent phases); here it hides behind the clearing.
template <bool DET>
__global__ void __launch_bounds__(GSR_TILE_ORDER_THREADS) k_backward_prologue(SurvLists surv, float* acc, uint8_t* aflag, int P, int clear_blocks,
                                                                              const uint32_t* __restrict__ work, uint32_t* __restrict__ order, int ntiles)
{
    const int first = (order != nullptr) ? 1 : 0;
    if ((int)blockIdx.x < first) {          // (block-uniform)
        tile_order_block(work, order, ntiles);
        return;
    }
    const uint32_t b = blockIdx.x - (uint32_t)first;
    if ((int)b >= clear_blocks) return;
    const uint32_t sl = b & (GSR_SURV_LISTS - 1);
    const uint32_t n = surv.n[sl * GSR_SURV_CSTRIDE];
    const uint32_t* __restrict__ list = surv.ids + (size_t)sl * surv.cap;
    const uint32_t step = ((uint32_t)clear_blocks / GSR_SURV_LISTS) * GSR_TILE_ORDER_THREADS;
    for (uint32_t c = (b / GSR_SURV_LISTS) * GSR_TILE_ORDER_THREADS + threadIdx.x; c < n; c += step) {
        const size_t idx = list[c];
        acc_clear<DET>(acc, idx);
        aflag[idx] = (uint8_t)0;
        aflag[(size_t)P + idx] = (uint8_t)0;
    }
}
template <bool DET>
__global__ void __launch_bounds__(64) k_preprocess_bwd(PreBwdArgs a)
{
    __shared__ float4 s_sh[GSR_K8_ROWS * GSR_SH16_LDS4];
    __shared__ uint32_t s_q[2 * GSR_K8_ROWS];      // queue of active Gaussians: index | has a colour gradient << 31
    __shared__ PoseStepLDS s_pose;
    const int lane = threadIdx.x;
    const bool frozen = a.guard.frozen();      // (a frozen iteration still takes its ticket: the last workgroup publishes the status)
    if (frozen && a.ticket == nullptr) return;
    // What this launch does (block-uniform; PreBwdArgs::role).  final_done is only ever written by the last workgroup of a launch,
    // after every workgroup has drawn its ticket: all workgroups of one launch read the same value.
    const bool conv = a.role == 1 && a.guard.conv != nullptr && *a.guard.conv != 0.f;
    // (rows_every: GSR_REFINE_GRADS_EVERY_ITERATION -- every iteration of the loop writes the rows itself, from its own set, like the
    // stateless backward; there is no final pass then.  Diagnostics: both ways must leave the same bits.)
    const bool every = a.rows_every != 0;
    const bool final_pass = !every && (a.role == 2 || conv) && *a.final_done == 0u;
    if (a.role == 2 && !final_pass) return;
    const bool walk = final_pass || !frozen;
    const bool rows_on = a.role == 0 || final_pass || every;      // gradient rows and dirty bits written, flags and records consumed
    const bool tau_on = a.pose != 0 && !final_pass;
    const bool clear_other = a.role == 1 && !conv && !every;       // (a poisoned group does this part too)
    const SurvLists wl = final_pass ? a.o_surv : a.surv;
    uint8_t* const wflag = final_pass ? a.o_aflag : a.aflag;
    float* const wacc = final_pass ? a.o_acc : a.acc;
    const float* const wrec = final_pass ? a.o_rec : a.rec;
    const uint8_t* const wclamped = final_pass ? a.o_clamped : a.clamped;
    const float* const view = final_pass ? a.o_cam : a.view;
    const float* const proj = final_pass ? a.o_cam + 16 : a.proj;
    const float* const campos = final_pass ? a.o_cam + 32 : a.campos;
    uint8_t* const dirty = rows_on ? a.dirty : nullptr;
    float* const o_dsh = rows_on ? a.dL_dsh : nullptr;
    // (the other set's list length, asked for up front: the wait for it hides behind the walk)
    const uint32_t rb = gridDim.x - 1u - blockIdx.x;      // reversed: the workgroups with chain-rule work sit at the front of the lists
    const uint32_t o_n = clear_other ? a.o_surv.n[(rb & (GSR_SURV_LISTS - 1)) * GSR_SURV_CSTRIDE] : 0u;
    float tw[12] = {0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0};      // world-frame sums behind dL/dtau, see (6) below
    long long twi[12] = {0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0};  // ... DET: in fixed point (which Gaussians share a lane depends on the lists' order)
    long long twn = 0;                                         // ... and how many terms were not finite (word 7 of the slot: the pose step reports NaN)
    GSR_T_DECL
  if (walk) {
    // SH rows in (and dL_dsh rows out) as 16-B-per-lane streams of whole 192-B rows through LDS
    const bool staged = (a.shs != nullptr) && sh16_vector_ok(a.M, a.shs) &&
                        (a.dL_dsh == nullptr || (reinterpret_cast<uintptr_t>(a.dL_dsh) & 15u) == 0);
    const GradRows rows = {a.dL_dmean2D, a.dL_dconic, a.dL_dopacity, a.dL_dcolor, a.dL_dmean3D, a.dL_dcov3D, a.dL_dsh, a.dL_dscale, a.dL_drot, a.M};
    const uint32_t sl = blockIdx.x & (GSR_SURV_LISTS - 1);
    const uint32_t n = wl.n[sl * GSR_SURV_CSTRIDE];
    const uint32_t* __restrict__ list = wl.ids + (size_t)sl * wl.cap;
    const uint32_t step = (gridDim.x / GSR_SURV_LISTS) * GSR_K8_ROWS;
    uint32_t c0 = (blockIdx.x / GSR_SURV_LISTS) * GSR_K8_ROWS;
    // (the first chunk of the list is requested together with the list's length -- inside the sub-list's allocation whatever the
    // length turns out to be -- instead of one round trip behind it)
    const uint32_t first_c0 = c0;
    const uint32_t first_entry = list[c0 + (uint32_t)lane];
    int qn = 0;          // active Gaussians queued in s_q (wave-uniform)
    for (;;) {
        // ---- fill: look at chunks of the list until 64 active Gaussians are queued (or the list ends).  A survivor nobody
        // blended has an all-zero record and all-zero gradients, whatever its other parameters are: on a long list (complete
        // bins: half of the survivors) the chain rule below would otherwise run on half-empty lanes.
        while (qn < GSR_K8_ROWS && c0 < n) {
            const bool in = c0 + (uint32_t)lane < n;
            const int idx = in ? (int)(c0 == first_c0 ? first_entry : list[c0 + lane]) : 0;
            c0 += step;
            // (round 4: the compositing backward flags the Gaussians it added anything to -- two bytes per survivor here instead of its
            // 48-byte record: complete lists make every visible Gaussian a survivor and nine in ten of them were never blended)
            const uint8_t fa = in ? wflag[idx] : (uint8_t)0, fc = in ? wflag[(size_t)a.P + idx] : (uint8_t)0;
            const bool active = fa != 0;
            // zero colour gradient => zero SH gradient whatever the coefficients are: their row is not even read
            const bool has_col = active && fc != 0;
            if (rows_on && fa != 0) wflag[idx] = (uint8_t)0;                       // consumed: clean for the next backward
            if (rows_on && fc != 0) wflag[(size_t)a.P + idx] = (uint8_t)0;
            // The gradient tensors are zero wherever nothing is written: the host zero-fills them per call, or (native
            // loop) once per frame, after which the dirty bits say which rows hold values from the iteration before.
            // (Rows of Gaussians that are not on this iteration's lists were cleared by k_preprocess.)
            const uint8_t was = (dirty != nullptr && in) ? dirty[idx] : (uint8_t)0;
            if (dirty != nullptr && in) {
                const uint8_t now = (uint8_t)((active ? 1 : 0) | (has_col ? 2 : 0));
                if (now != was) dirty[idx] = now;
            }
            if (!active && (was & 1)) zero_grad_rows(rows, (size_t)idx, true, false);      // no gradient any more
            if ((was & 2) && !has_col) zero_grad_rows(rows, (size_t)idx, false, true);       // had an SH gradient last iteration, has none now
            const unsigned long long mk = __ballot(active);
            if (active) s_q[qn + (int)__popcll(mk & ((1ull << lane) - 1ull))] = (uint32_t)idx | (has_col ? 0x80000000u : 0u);
            qn += (int)__popcll(mk);
        }
        GSR_T_TICK(0)
        if (qn == 0) break;
        __syncthreads();
        GSR_T_COUNT(10, 1)
        // ---- chain rule on the first (up to) 64 queued Gaussians, dense lanes (their records are re-read: L2 hits)
        const int nrow = min(qn, GSR_K8_ROWS);
        const bool active = lane < nrow;
        const uint32_t qe = active ? s_q[lane] : 0u;
        const int idx = (int)(qe & 0x7FFFFFFFu);
        const bool has_col = (qe >> 31) != 0u;
        float4 r0 = make_float4(0.f, 0.f, 0.f, 0.f), r1 = r0, r2 = r0;
        if (active) {
            acc_load<DET>(wacc, (size_t)idx, r0, r1, r2);
            if (dirty != nullptr) acc_clear<DET>(wacc, (size_t)idx);      // native loop, final pass: leave the record clean for the next call's K7 (no 48 MB memset)
            if (rows_on) {
                a.dL_dcolor[3 * (size_t)idx] = r0.x; a.dL_dcolor[3 * (size_t)idx + 1] = r0.y; a.dL_dcolor[3 * (size_t)idx + 2] = r0.z;
                a.dL_dmean2D[3 * (size_t)idx] = r0.w; a.dL_dmean2D[3 * (size_t)idx + 1] = r1.x;
                reinterpret_cast<float4*>(a.dL_dconic)[idx] = make_float4(r1.y, r1.z, 0.f, r1.w);
                a.dL_dopacity[idx] = r2.x;
            }
        }
        const unsigned long long colmask = __ballot(has_col);
        // Every per-Gaussian read of the round is requested here, in FRONT of the SH rows, so that one round trip covers them all
        // (the rows' LDS stores wait for the last loads issued; round 2 asked for these after the barrier below: a second trip).
        float cov6[6] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        float3 mean = make_float3(0.f, 0.f, 0.f);
        SplatRec sr = {};
        const bool want_sr = rows_on && a.scales && (a.dL_dscale || a.dL_drot);
        float s3[3] = {0.f, 0.f, 0.f};
        float4 q = make_float4(0.f, 0.f, 0.f, 0.f);
        if (active) {
#pragma unroll
            for (int i = 0; i < 6; i++) cov6[i] = a.cov3D[6 * (size_t)idx + i];
            mean = make_float3(a.means[3 * idx], a.means[3 * idx + 1], a.means[3 * idx + 2]);
            sr = load_splat_rec(wrec, (uint32_t)idx);
            if (want_sr) {
                s3[0] = a.scales[3 * idx]; s3[1] = a.scales[3 * idx + 1]; s3[2] = a.scales[3 * idx + 2];
                q = reinterpret_cast<const float4*>(a.rots)[idx];
            }
        }
        if (staged) {
#pragma unroll
            for (int i = 0; i < GSR_SH16_ROW4; i++) {
                const int j = lane + 64 * i;
                const int r = j / GSR_SH16_ROW4, part = j - r * GSR_SH16_ROW4;
                const int rid = __shfl(idx, r, 64);
                if ((colmask >> r) & 1ull)
                    s_sh[r * GSR_SH16_LDS4 + part] = reinterpret_cast<const float4*>(a.shs)[(size_t)rid * GSR_SH16_ROW4 + part];
            }
        }
        __syncthreads();
        GSR_T_TICK(1)
        GSR_T_COUNT(11, nrow)
        float* my_row = reinterpret_cast<float*>(&s_sh[lane * GSR_SH16_LDS4]);
        if (active) {
            const float3 co = make_float3(sr.a, sr.b, sr.c);
            // (1) conic gradient -> covariance gradient and the mean's share through the projected covariance
            float G[6];
            const float3 g_cov = covariance_chain(mean, cov6, make_float3(co.x, co.y, co.z), make_float3(r1.y, r1.z, r1.w), view, a.fx, a.fy,
                                                  a.tanx, a.tany, G);
            if (rows_on && a.dL_dcov3D) {      // the reference's 6-vector counts each off-diagonal entry twice
                float* o = a.dL_dcov3D + 6 * (size_t)idx;
                o[0] = G[0]; o[1] = 2.f * G[1]; o[2] = 2.f * G[2]; o[3] = G[3]; o[4] = 2.f * G[4]; o[5] = G[5];
            }
            // (2) screen-space mean gradient through the perspective division (backward.cu:346-372)
            const float* P = proj;
            const float hx = P[0] * mean.x + P[4] * mean.y + P[8] * mean.z + P[12], hy = P[1] * mean.x + P[5] * mean.y + P[9] * mean.z + P[13];
            const float hw = P[3] * mean.x + P[7] * mean.y + P[11] * mean.z + P[15];
            const float rw = 1.0f / (hw + 0.0000001f);
            const float kx = hx * rw * rw, ky = hy * rw * rw, g2x = r0.w, g2y = r1.x;
            const float3 g_m2d = make_float3((P[0] * rw - P[3] * kx) * g2x + (P[1] * rw - P[3] * ky) * g2y,
                                             (P[4] * rw - P[7] * kx) * g2x + (P[5] * rw - P[7] * ky) * g2y,
                                             (P[8] * rw - P[11] * kx) * g2x + (P[9] * rw - P[11] * ky) * g2y);
            // (3) pose package: the splat's own depth z = (Wc p + trans).z carries gradient too
            float3 g_geo = make_float3(g_cov.x + g_m2d.x, g_cov.y + g_m2d.y, g_cov.z + g_m2d.z);
            if (a.pose) {
                const float dz = r2.y;
                g_geo.x += view[2] * dz; g_geo.y += view[6] * dz; g_geo.z += view[10] * dz;
            }
            GSR_T_TICK(2)
            // (4) colour gradient -> SH coefficients and the view direction's share of the mean gradient
            float3 g_sh = make_float3(0.f, 0.f, 0.f);
            if (a.shs && has_col) {
                const float3 dcol = make_float3(r0.x, r0.y, r0.z);
                if (staged)
                    g_sh = sh_color_backward(a.D, 16, mean, campos, my_row, wclamped[idx], dcol, o_dsh ? my_row : nullptr);
                else
                    g_sh = sh_color_backward(a.D, a.M, mean, campos, a.shs + (size_t)idx * a.M * 3, wclamped[idx], dcol,
                                             o_dsh ? o_dsh + (size_t)idx * a.M * 3 : nullptr);
            }
            GSR_T_TICK(3)
            if (rows_on && a.dL_dmean3D) {
                a.dL_dmean3D[3 * (size_t)idx] = g_geo.x + g_sh.x;
                a.dL_dmean3D[3 * (size_t)idx + 1] = g_geo.y + g_sh.y;
                a.dL_dmean3D[3 * (size_t)idx + 2] = g_geo.z + g_sh.z;
            }
            // (5) covariance gradient -> scale and quaternion
            if (want_sr) {
                float ds[3], dq[4];
                covariance_param_grads(s3, a.mod, q, G, ds, dq);
                if (a.dL_dscale) {
                    a.dL_dscale[3 * (size_t)idx] = ds[0]; a.dL_dscale[3 * (size_t)idx + 1] = ds[1]; a.dL_dscale[3 * (size_t)idx + 2] = ds[2];
                }
                if (a.dL_drot) reinterpret_cast<float4*>(a.dL_drot)[idx] = make_float4(dq[0], dq[1], dq[2], dq[3]);
            }
            // (6) pose package: dL/dtau for T_w2c <- exp([rho, theta]) T_w2c at 0.  With
            //   p_C = Wc p + trans:  drho = Wc (g_geo + g_sh),  dtheta = p_C x (Wc g_geo) + 2 Wc a,
            //   a = (X_12, X_20, X_01) of the antisymmetric X = Sigma G - G Sigma (how the covariance turns with the camera).
            // Everything per Gaussian is kept in the WORLD frame -- p_C x (Wc g) = Wc (p x g) + trans x (Wc g) -- and the
            // rotation is applied once per wave to the sums (tw: rho part, g_geo, p x g_geo, a).
            if (tau_on) {
                // P = Sigma G; X_ij = P_ij - P_ji
                const float P01 = cov6[0] * G[1] + cov6[1] * G[3] + cov6[2] * G[4], P10 = cov6[1] * G[0] + cov6[3] * G[1] + cov6[4] * G[2];
                const float P02 = cov6[0] * G[2] + cov6[1] * G[4] + cov6[2] * G[5], P20 = cov6[2] * G[0] + cov6[4] * G[1] + cov6[5] * G[2];
                const float P12 = cov6[1] * G[2] + cov6[3] * G[4] + cov6[4] * G[5], P21 = cov6[2] * G[1] + cov6[4] * G[3] + cov6[5] * G[4];
                const float term[12] = {g_geo.x + g_sh.x, g_geo.y + g_sh.y, g_geo.z + g_sh.z, g_geo.x, g_geo.y, g_geo.z,
                                        mean.y * g_geo.z - mean.z * g_geo.y, mean.z * g_geo.x - mean.x * g_geo.z, mean.x * g_geo.y - mean.y * g_geo.x,
                                        2.f * (P12 - P21), 2.f * (P20 - P02), 2.f * (P01 - P10)};
#pragma unroll
                for (int i = 0; i < 12; i++) {
                    if (DET) { if (__builtin_isfinite(term[i])) twi[i] += to_fixed(term[i], GSR_FIX_TAU); else twn++; }
                    else tw[i] += term[i];
                }
            }
        }
        GSR_T_TICK(4)
        if (staged && o_dsh) {
            __syncthreads();
#pragma unroll
            for (int i = 0; i < GSR_SH16_ROW4; i++) {
                const int j = lane + 64 * i;
                const int r = j / GSR_SH16_ROW4, part = j - r * GSR_SH16_ROW4;
                const int rid = __shfl(idx, r, 64);
                if ((colmask >> r) & 1ull)
                    reinterpret_cast<float4*>(o_dsh)[(size_t)rid * GSR_SH16_ROW4 + part] = s_sh[r * GSR_SH16_LDS4 + part];
            }
        }
        // the rest of the queue moves to the front
        const uint32_t keep = (nrow + lane < qn) ? s_q[nrow + lane] : 0u;
        __syncthreads();
        if (nrow + lane < qn) s_q[lane] = keep;
        qn -= nrow;
        __syncthreads();
        GSR_T_TICK(5)
    }
    if (tau_on) {
        // wave reduction in fp64, rotation into the camera frame, then one fp64 atomic per wave and component into one of
        // GSR_TAU_SLOTS partial sums (64 B apart: thousands of waves adding into six words would queue up at the memory-side atomic unit)
        // (a wave that queued nothing -- seven in eight of them in a speculative iteration -- has nothing to add)
        bool any = false;
#pragma unroll
        for (int i = 0; i < 12; i++) any = any || (DET ? twi[i] != 0 : tw[i] != 0.f);
        if (DET) any = any || (twn != 0);
        const bool wave_any = __ballot(any) != 0ull;          // (wave-uniform; evaluated by all lanes, outside the lane-63 branch below)
        double sw[12];
        if (DET && wave_any) {
            // deterministic option: the twelve world-frame sums themselves leave the wave, as integers (the pose step rotates the totals)
            unsigned long long* ta = reinterpret_cast<unsigned long long*>(a.tau_acc) + (blockIdx.x & (GSR_TAU_SLOTS - 1)) * 8;
#pragma unroll
            for (int i = 0; i < 12; i++) {
                const long long t = wave_sum_ll_to_lane63(twi[i]);
                if (lane == 63 && t != 0) atomicAdd(&ta[(i < 6 ? 0 : 8 * GSR_TAU_SLOTS) + (i < 6 ? i : i - 6)], (unsigned long long)t);
            }
            const long long tn = wave_sum_ll_to_lane63(twn);
            if (lane == 63 && tn != 0) atomicAdd(&ta[7], (unsigned long long)tn);
        }
        if (!DET && wave_any) {
#pragma unroll
            for (int i = 0; i < 12; i++) sw[i] = wave_sum_d_to_lane63((double)tw[i]);
        }
        if (!DET && lane == 63 && wave_any) {
            const float* vm = view;
            double tau[6], wg[3];
#pragma unroll
            for (int r = 0; r < 3; r++) {
                const double w0 = vm[r], w1 = vm[4 + r], w2 = vm[8 + r];          // row r of Wc
                tau[r] = w0 * sw[0] + w1 * sw[1] + w2 * sw[2];
                wg[r] = w0 * sw[3] + w1 * sw[4] + w2 * sw[5];
                tau[3 + r] = w0 * (sw[6] + sw[9]) + w1 * (sw[7] + sw[10]) + w2 * (sw[8] + sw[11]);
            }
            const double t0 = vm[12], t1 = vm[13], t2 = vm[14];
            tau[3] += t1 * wg[2] - t2 * wg[1]; tau[4] += t2 * wg[0] - t0 * wg[2]; tau[5] += t0 * wg[1] - t1 * wg[0];
#pragma unroll
            for (int i = 0; i < 6; i++)
                if (tau[i] != 0.0) atomicAdd(&a.tau_acc[(blockIdx.x & (GSR_TAU_SLOTS - 1)) * 8 + i], tau[i]);
        }
    }
    GSR_T_TICK(6)
  }
    if (clear_other) {
        // what the group in front of this one left in ITS set: flags and records of the Gaussians its compositing backward added to
        // (this group's own compositing backward has run on the other set; the next group's will run on this one)
        const uint32_t* __restrict__ list2 = a.o_surv.ids + (size_t)(rb & (GSR_SURV_LISTS - 1)) * a.o_surv.cap;
        const uint32_t step2 = (gridDim.x / GSR_SURV_LISTS) * GSR_K8_ROWS;
        for (uint32_t c = (rb / GSR_SURV_LISTS) * GSR_K8_ROWS; c < o_n; c += step2) {
            if (c + (uint32_t)lane < o_n) {
                const size_t idx = list2[c + (uint32_t)lane];
                const uint8_t fa = a.o_aflag[idx], fc = a.o_aflag[(size_t)a.P + idx];
                if (fa != 0) { a.o_aflag[idx] = (uint8_t)0; acc_clear<DET>(a.o_acc, idx); }
                if (fc != 0) a.o_aflag[(size_t)a.P + idx] = (uint8_t)0;
            }
        }
    }
    if (a.ticket != nullptr) {
        // Two levels: ~2000 workgroups drawing from ONE counter would queue up at the memory-side atomic unit for longer
        // than the kernel runs (measured: +54 us).  Workgroups sharing a dL/dtau slot (blockIdx mod 64) count in the unused
        // words of that slot; the last of each group draws from the main ticket.  (The pose step zeroes the slots.)
        const uint32_t grp = blockIdx.x & (GSR_TAU_SLOTS - 1);
        const uint32_t in_grp = (gridDim.x - grp + GSR_TAU_SLOTS - 1) / GSR_TAU_SLOTS;
        const uint32_t ngrp = min((uint32_t)GSR_TAU_SLOTS, gridDim.x);
        // The dL/dtau sums are memory-side atomics: once they have completed (vmcnt drained) every later reader sees them --
        // no release fence, which at agent scope would write this XCD's whole L2 back (measured: +50 us on this kernel).
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        uint32_t t = 0u;
        if (lane == 0) {
            t = atomicAdd(reinterpret_cast<uint32_t*>(&a.tau_acc[grp * 8 + 6]), 1u);
            if (t == in_grp - 1u) t = atomicAdd(a.ticket, 1u) + 0x10000u;
        }
        t = (uint32_t)__builtin_amdgcn_readfirstlane((int)t);
        GSR_T_TICK(7)
        if (t == 0x10000u + ngrp - 1u) {
            // last of all: everybody's sums are in (read below with agent-scope atomic loads, past this CU's L1)
            if (lane == 0) *a.ticket = 0u;             // (the next launch starts counting from zero)
            reinterpret_cast<uint32_t*>(&a.tau_acc[lane * 8 + 6])[0] = 0u;      // the group counters too, also on a frozen iteration
            // every workgroup is past the other set's work list, which holds nothing any more: the forward after next appends from zero
            // (role 1 is the only one with a ticket; the own set's counters are returned by the next group's launch)
            a.o_surv.n[lane * GSR_SURV_CSTRIDE] = 0u;
            if (final_pass && lane == 0) *a.final_done = 1u;
            pose_step_wave<DET>(a.fold, a.guard, s_pose);
            GSR_T_TICK(8)
        }
    }
    GSR_T_FLUSH(48)
}

__device__ __forceinline__ double tau_total(const double* acc, int i)
{
    double t = 0.0;
    for (int sl = 0; sl < GSR_TAU_SLOTS; sl++) t += acc[sl * 8 + i];
    return t;
}
__global__ void k_tau_finish(const double* acc, float* out)
{
    if (threadIdx.x < 6) out[threadIdx.x] = (float)tau_total(acc, threadIdx.x);
}
// deterministic option: the slots hold the twelve fixed-point world-frame sums (k_preprocess_bwd<true>); one wave, lane = slot
__global__ void __launch_bounds__(64) k_tau_finish_det(const long long* acc, const float* view, float* out)
{
    const int lane = threadIdx.x;
    double sw[12];
#pragma unroll
    for (int i = 0; i < 12; i++)
        sw[i] = from_fixed(wave_sum_ll_to_lane63(acc[(i < 6 ? 0 : 8 * GSR_TAU_SLOTS) + lane * 8 + (i < 6 ? i : i - 6)]), GSR_FIX_TAU);
    const long long nonfinite = wave_sum_ll_to_lane63(acc[lane * 8 + 7]);
    if (lane == 63) {
        float vm[16];
        for (int k = 0; k < 16; k++) vm[k] = view[k];
        double tau[6];
        tau_from_world_sums(sw, vm, tau);
        for (int i = 0; i < 6; i++) out[i] = (nonfinite != 0) ? __builtin_nanf("") : (float)tau[i];
    }
}

// ---------------------------------------------------------------------------------------------
// distCUDA2: mean squared distance of every point to its three nearest neighbours,
// gaussian_splatting/submodules/simple-knn/simple_knn.cu:45-220 (the only native dependency of create_from_pcd).
// Same plan as the reference -- Morton order, axis-aligned boxes over runs of 1024 sorted points, exact search
// with box pruning -- re-cut for wave64: the points are first GATHERED into Morton order (float4, original index
// in .w) so that a wave's 64 points are spatial neighbours; the wave tests each box ONCE against its own bounding
// box and current search radius, and a surviving box's points are read at wave-uniform addresses (scalar loads,
// broadcast to all lanes), each lane keeping its own three best.  The pruning is conservative at both levels,
// so the result is the exact 3-NN mean like the reference's.
// ---------------------------------------------------------------------------------------------
#define GSR_KNN_BOX 1024
__device__ __forceinline__ uint32_t knn_prep_morton(uint32_t x)
{
    x = (x | (x << 16)) & 0x030000FFu;
    x = (x | (x << 8)) & 0x0300F00Fu;
    x = (x | (x << 4)) & 0x030C30C3u;
    x = (x | (x << 2)) & 0x09249249u;
    return x;
}
// min / max over all points, seeded with the origin like the reference's reductions (simple_knn.cu:184-194,
// init = {0,0,0}); floats are compared through an order-preserving integer encoding
__device__ __forceinline__ uint32_t f2ord(float f) { const uint32_t b = __float_as_uint(f); return (b & 0x80000000u) ? ~b : (b | 0x80000000u); }
__device__ __forceinline__ float ord2f(uint32_t u) { return __uint_as_float((u & 0x80000000u) ? (u & 0x7FFFFFFFu) : ~u); }
__global__ void __launch_bounds__(GSR_BLOCK) k_knn_minmax(int P, const float* __restrict__ pts, uint32_t* __restrict__ mm /*[6]: min xyz, max xyz (encoded)*/)
{
    float lo[3] = {0.f, 0.f, 0.f}, hi[3] = {0.f, 0.f, 0.f};
    for (int i = blockIdx.x * GSR_BLOCK + threadIdx.x; i < P; i += gridDim.x * GSR_BLOCK)
#pragma unroll
        for (int c = 0; c < 3; c++) { const float v = pts[3 * (size_t)i + c]; lo[c] = fminf(lo[c], v); hi[c] = fmaxf(hi[c], v); }
#pragma unroll
    for (int c = 0; c < 3; c++) {
#pragma unroll
        for (int off = 32; off > 0; off >>= 1) { lo[c] = fminf(lo[c], __shfl_xor(lo[c], off, 64)); hi[c] = fmaxf(hi[c], __shfl_xor(hi[c], off, 64)); }
        if ((threadIdx.x & 63) == 0) { atomicMin(&mm[c], f2ord(lo[c])); atomicMax(&mm[3 + c], f2ord(hi[c])); }
    }
}
__global__ void __launch_bounds__(GSR_BLOCK) k_knn_morton(int P, const float* __restrict__ pts, const uint32_t* __restrict__ mm,
                                                          uint32_t* __restrict__ codes, uint32_t* __restrict__ idx)
{
    const int i = blockIdx.x * GSR_BLOCK + threadIdx.x;
    if (i >= P) return;
    uint32_t code = 0;
#pragma unroll
    for (int c = 0; c < 3; c++) {
        const float lo = ord2f(mm[c]), hi = ord2f(mm[3 + c]);
        const float t = ((pts[3 * (size_t)i + c] - lo) / (hi - lo)) * (float)((1 << 10) - 1);      // simple_knn.cu:57-66
        code |= knn_prep_morton((uint32_t)t) << c;
    }
    codes[i] = code;
    idx[i] = (uint32_t)i;
}
__global__ void __launch_bounds__(GSR_BLOCK) k_knn_gather(int P, const float* __restrict__ pts, const uint32_t* __restrict__ idx_sorted,
                                                          float4* __restrict__ sorted)
{
    const int i = blockIdx.x * GSR_BLOCK + threadIdx.x;
    if (i >= P) return;
    const uint32_t j = idx_sorted[i];
    sorted[i] = make_float4(pts[3 * (size_t)j], pts[3 * (size_t)j + 1], pts[3 * (size_t)j + 2], __uint_as_float(j));
}
// one workgroup of 1024 lanes per box (simple_knn.cu:83-123)
__global__ void __launch_bounds__(GSR_KNN_BOX) k_knn_boxes(int P, const float4* __restrict__ sorted, float* __restrict__ boxes /*[nb][8]*/)
{
    __shared__ float s_lo[16][3], s_hi[16][3];
    const int i = blockIdx.x * GSR_KNN_BOX + threadIdx.x;
    float lo[3] = {3.402823466e38f, 3.402823466e38f, 3.402823466e38f}, hi[3] = {-3.402823466e38f, -3.402823466e38f, -3.402823466e38f};
    if (i < P) { const float4 p = sorted[i]; lo[0] = hi[0] = p.x; lo[1] = hi[1] = p.y; lo[2] = hi[2] = p.z; }
#pragma unroll
    for (int c = 0; c < 3; c++) {
#pragma unroll
        for (int off = 32; off > 0; off >>= 1) { lo[c] = fminf(lo[c], __shfl_xor(lo[c], off, 64)); hi[c] = fmaxf(hi[c], __shfl_xor(hi[c], off, 64)); }
        if ((threadIdx.x & 63) == 0) { s_lo[threadIdx.x >> 6][c] = lo[c]; s_hi[threadIdx.x >> 6][c] = hi[c]; }
    }
    __syncthreads();
    if (threadIdx.x < 3) {
        float l = s_lo[0][threadIdx.x], h = s_hi[0][threadIdx.x];
        for (int w = 1; w < 16; w++) { l = fminf(l, s_lo[w][threadIdx.x]); h = fmaxf(h, s_hi[w][threadIdx.x]); }
        boxes[blockIdx.x * 8 + threadIdx.x] = l; boxes[blockIdx.x * 8 + 4 + threadIdx.x] = h;
    }
}
__device__ __forceinline__ void knn_update3(float dist, float* best)      // simple_knn.cu:137-151
{
#pragma unroll
    for (int j = 0; j < 3; j++)
        if (best[j] > dist) { const float t = best[j]; best[j] = dist; dist = t; }
}
__device__ __forceinline__ float knn_dist2(float4 a, float4 b)
{
    const float dx = b.x - a.x, dy = b.y - a.y, dz = b.z - a.z;
    return dx * dx + dy * dy + dz * dz;
}
__global__ void __launch_bounds__(GSR_BLOCK) k_knn_search(int P, const float4* __restrict__ sorted, const float* __restrict__ boxes,
                                                          int nboxes, float* __restrict__ dists)
{
    const int lane = threadIdx.x & 63;
    const int w0 = (blockIdx.x * GSR_BLOCK + (threadIdx.x & ~63));        // first sorted index of this wave
    if (w0 >= P) return;
    const int i = w0 + lane;
    const bool live = i < P;
    const float4 me = sorted[live ? i : P - 1];
    const float FMAX = 3.402823466e38f;
    float best[3] = {FMAX, FMAX, FMAX};
    if (live)
        for (int k = max(0, i - 3); k <= min(P - 1, i + 3); k++)
            if (k != i) knn_update3(knn_dist2(me, sorted[k]), best);
    const float reject = best[2];                          // an upper bound of the third-nearest distance
    best[0] = FMAX; best[1] = FMAX; best[2] = FMAX;
    // the wave's own bounding box
    float lo[3] = {live ? me.x : FMAX, live ? me.y : FMAX, live ? me.z : FMAX}, hi[3] = {live ? me.x : -FMAX, live ? me.y : -FMAX, live ? me.z : -FMAX};
#pragma unroll
    for (int c = 0; c < 3; c++)
#pragma unroll
        for (int off = 32; off > 0; off >>= 1) { lo[c] = fminf(lo[c], __shfl_xor(lo[c], off, 64)); hi[c] = fmaxf(hi[c], __shfl_xor(hi[c], off, 64)); }
    for (int b = 0; b < nboxes; b++) {
        const float bl[3] = {boxes[b * 8], boxes[b * 8 + 1], boxes[b * 8 + 2]}, bh[3] = {boxes[b * 8 + 4], boxes[b * 8 + 5], boxes[b * 8 + 6]};
        // wave level: squared gap between the two boxes against the largest radius any lane still searches
        float rad = live ? fminf(reject, best[2]) : 0.f;
#pragma unroll
        for (int off = 32; off > 0; off >>= 1) rad = fmaxf(rad, __shfl_xor(rad, off, 64));
        float gap = 0.f;
#pragma unroll
        for (int c = 0; c < 3; c++) { const float g = fmaxf(0.f, fmaxf(bl[c] - hi[c], lo[c] - bh[c])); gap += g * g; }
        if (gap > rad) continue;                           // wave-uniform
        // lane level: the reference's own test (simple_knn.cu:125-135, 177-180)
        float d2 = 0.f;
        {
            const float p3[3] = {me.x, me.y, me.z};
#pragma unroll
            for (int c = 0; c < 3; c++)
                if (p3[c] < bl[c] || p3[c] > bh[c]) { const float g = fminf(fabsf(p3[c] - bl[c]), fabsf(p3[c] - bh[c])); d2 += g * g; }
        }
        const bool want = live && !(d2 > reject || d2 > best[2]);
        if (__ballot(want) == 0ull) continue;
        const int e = min(P, (b + 1) * GSR_KNN_BOX);
        for (int k = b * GSR_KNN_BOX; k < e; k++) {
            const float4 q = sorted[k];                    // wave-uniform address: one scalar load for all lanes
            if (want && k != i) knn_update3(knn_dist2(me, q), best);
        }
    }
    if (live) dists[__float_as_uint(me.w)] = (best[0] + best[1] + best[2]) / 3.0f;
}

// ---------------------------------------------------------------------------------------------
// Training-step loss epilogue: gaussian_splatting/train.py:92-108 with
// utils/loss_utils.py:17-63 and their autograd backward, as four launches instead of ~60:
//   loss = (1 - lambda) L1(image, gt) + lambda (1 - SSIM(image, gt)) + w_d min(1 - rho(-m, d), 1 - rho(1/(m+200), d))
// SSIM: 11x11 Gaussian window (sigma 1.5), zero padding, per channel.  Every statistic of _ssim is a window
// filter of x, y, xx, yy, xy, so the map is a function F(mu1, mu2, Exx, Eyy, Exy) per pixel and
//   dSSIM/dx(q) = sum_p w(p - q) [ F_mu1(p) + 2 x(q) F_Exx(p) + y(q) F_Exy(p) ] / (3N):
// pass 1 (k_ssim_fwd) filters the five inputs (separable, 42x42 halo tile in LDS), evaluates the map, sums it
// and the L1 term, and stores the three partial-derivative maps; pass 2 (k_ssim_bwd) filters those maps with
// the same (symmetric) window and assembles dL/dimage including the L1 sign term.  HBM traffic per pixel and
// channel: 8 B in + 12 B out, then 12 B + 8 B in + 4 B out.
// ---------------------------------------------------------------------------------------------
#define GSR_SSIM_R 5
#define GSR_SSIM_T 32                                  // output tile: 32 x 32 pixels per workgroup of 256 lanes, four pixels per lane
#define GSR_SSIM_H (GSR_SSIM_T + 2 * GSR_SSIM_R)      // 42
#define GSR_SSIM_S (GSR_SSIM_H + 2)                    // row stride of the staged halo tile (16-byte aligned rows)
#define GSR_SSIM_THREADS 256
struct SsimArgs {
    int W, H;
    const float* img; const float* gt;       // [3, H, W]
    float lambda_dssim;
    float* maps;                             // workspace: [3 maps][3 channels][H][W]  (F_mu1, F_Exx, F_Exy)
    double* sums;                            // [0] sum |x - y|, [1] sum ssim_map   (fp64 atomics)
    float* dL_dimage;
    float w[2 * GSR_SSIM_R + 1];             // gaussian(11, 1.5), normalised (loss_utils.py:23-25)
};
// Round 4: 16 x 16 tiles with one pixel per lane took 169 us at 1296 x 840 (595 vector instructions per wave, 2.6x halo reads, every
// tap an LDS read).  Now 32 x 32 tiles: the horizontal pass hands a lane FOUR neighbouring outputs of a halo row -- 14 inputs read
// once (vector LDS reads), their squares and product formed once -- and the vertical pass four neighbouring rows of a column (14
// LDS reads per quantity for 44 FMAs).  Sums are taken in the same tap order as before (k = 0 ... 10), so every map value keeps its bits.
#define GSR_SSIM_HPASS(NQ, LOAD14, STORE)                                                                                    \
    for (int it = tid; it < GSR_SSIM_H * (GSR_SSIM_T / 4); it += GSR_SSIM_THREADS) {                                         \
        const int r = it / (GSR_SSIM_T / 4), c0 = 4 * (it - r * (GSR_SSIM_T / 4));                                           \
        float in[NQ][14];                                                                                                    \
        LOAD14                                                                                                               \
        float acc[NQ][4];                                                                                                    \
        _Pragma("unroll") for (int q = 0; q < NQ; q++)                                                                       \
            _Pragma("unroll") for (int o = 0; o < 4; o++) {                                                                  \
                float t = 0.f;                                                                                               \
                _Pragma("unroll") for (int k = 0; k < 2 * GSR_SSIM_R + 1; k++) t += a.w[k] * in[q][o + k];                   \
                acc[q][o] = t;                                                                                               \
            }                                                                                                                \
        STORE                                                                                                                \
    }

__global__ void __launch_bounds__(GSR_SSIM_THREADS) k_ssim_fwd(SsimArgs a)
{
    __shared__ __attribute__((aligned(16))) float s_x[GSR_SSIM_H][GSR_SSIM_S], s_y[GSR_SSIM_H][GSR_SSIM_S];
    __shared__ __attribute__((aligned(16))) float s_h[5][GSR_SSIM_H][GSR_SSIM_T];       // horizontally filtered x, y, xx, yy, xy
    __shared__ double s_red[4][2];
    const int tid = threadIdx.x;
    const int ch = blockIdx.z;
    const int x0 = blockIdx.x * GSR_SSIM_T, y0 = blockIdx.y * GSR_SSIM_T;
    const size_t N = (size_t)a.W * a.H;
    const float* img = a.img + ch * N;
    const float* gt = a.gt + ch * N;
    for (int i = tid; i < GSR_SSIM_H * GSR_SSIM_H; i += GSR_SSIM_THREADS) {
        const int r = i / GSR_SSIM_H, c = i - r * GSR_SSIM_H;
        const int gx = x0 + c - GSR_SSIM_R, gy = y0 + r - GSR_SSIM_R;
        const bool in = gx >= 0 && gx < a.W && gy >= 0 && gy < a.H;          // zero padding (F.conv2d padding = 5)
        s_x[r][c] = in ? img[(size_t)gy * a.W + gx] : 0.f;
        s_y[r][c] = in ? gt[(size_t)gy * a.W + gx] : 0.f;
    }
    __syncthreads();
    // (in[0] = x, in[1] = y, in[2] = xx, in[3] = yy, in[4] = xy over the lane's 14 halo columns)
#define GSR_SSIM_LOAD_FWD                                                                                                    \
        _Pragma("unroll") for (int v = 0; v < 3; v++) {                                                                      \
            const float4 xv = *reinterpret_cast<const float4*>(&s_x[r][c0 + 4 * v]);                                        \
            const float4 yv = *reinterpret_cast<const float4*>(&s_y[r][c0 + 4 * v]);                                        \
            in[0][4 * v] = xv.x; in[0][4 * v + 1] = xv.y; in[0][4 * v + 2] = xv.z; in[0][4 * v + 3] = xv.w;                  \
            in[1][4 * v] = yv.x; in[1][4 * v + 1] = yv.y; in[1][4 * v + 2] = yv.z; in[1][4 * v + 3] = yv.w;                  \
        }                                                                                                                    \
        { const float2 xv = *reinterpret_cast<const float2*>(&s_x[r][c0 + 12]); in[0][12] = xv.x; in[0][13] = xv.y;          \
          const float2 yv = *reinterpret_cast<const float2*>(&s_y[r][c0 + 12]); in[1][12] = yv.x; in[1][13] = yv.y; }        \
        _Pragma("unroll") for (int j = 0; j < 14; j++) {                                                                     \
            in[2][j] = in[0][j] * in[0][j]; in[3][j] = in[1][j] * in[1][j]; in[4][j] = in[0][j] * in[1][j];                  \
        }
#define GSR_SSIM_STORE5                                                                                                      \
        _Pragma("unroll") for (int q = 0; q < 5; q++)                                                                        \
            *reinterpret_cast<float4*>(&s_h[q][r][c0]) = make_float4(acc[q][0], acc[q][1], acc[q][2], acc[q][3]);
    GSR_SSIM_HPASS(5, GSR_SSIM_LOAD_FWD, GSR_SSIM_STORE5)
#undef GSR_SSIM_LOAD_FWD
#undef GSR_SSIM_STORE5
    __syncthreads();
    // vertical pass: lane = column lx, rows 4 ly ... 4 ly + 3
    const int lx = tid & (GSR_SSIM_T - 1), ly = tid >> 5;
    float f[5][4];
#pragma unroll
    for (int q = 0; q < 5; q++) {
        float col[14];
#pragma unroll
        for (int j = 0; j < 14; j++) col[j] = s_h[q][4 * ly + j][lx];
#pragma unroll
        for (int o = 0; o < 4; o++) {
            float t = 0.f;
#pragma unroll
            for (int k = 0; k < 2 * GSR_SSIM_R + 1; k++) t += a.w[k] * col[o + k];
            f[q][o] = t;
        }
    }
    const int px = x0 + lx;
    double l1 = 0.0, ss = 0.0;
#pragma unroll
    for (int o = 0; o < 4; o++) {
        const int py = y0 + 4 * ly + o;
        if (px < a.W && py < a.H) {
            const float mu1 = f[0][o], mu2 = f[1][o], exx = f[2][o], eyy = f[3][o], exy = f[4][o];
            const float C1 = 0.01f * 0.01f, C2 = 0.03f * 0.03f;
            const float mu1_sq = mu1 * mu1, mu2_sq = mu2 * mu2, mu12 = mu1 * mu2;
            const float s1 = exx - mu1_sq, s2 = eyy - mu2_sq, s12 = exy - mu12;
            const float A = 2.f * mu12 + C1, B = 2.f * s12 + C2, Cd = mu1_sq + mu2_sq + C1, D = s1 + s2 + C2;
            const float inv = 1.f / (Cd * D);
            const float ssim = A * B * inv;
            // F(mu1, mu2, Exx, Eyy, Exy) with s1 = Exx - mu1^2, s12 = Exy - mu1 mu2:
            //   dF/dExx = -A B / (Cd D^2),  dF/dExy = 2 A / (Cd D),
            //   dF/dmu1 = 2 mu2 B/(Cd D) - 2 mu2 A/(Cd D) ... collected below (chain through s1 and s12 included)
            const float F_exx = -ssim / D;
            const float F_exy = 2.f * A * inv;
            const float F_mu1 = 2.f * mu2 * B * inv - 2.f * mu1 * ssim / Cd - 2.f * mu1 * F_exx - mu2 * F_exy;
            const size_t o_ = ch * N + (size_t)py * a.W + px;
            a.maps[o_] = F_mu1; a.maps[3 * N + o_] = F_exx; a.maps[6 * N + o_] = F_exy;
            ss += (double)ssim;
            l1 += (double)fabsf(s_x[4 * ly + o + GSR_SSIM_R][lx + GSR_SSIM_R] - s_y[4 * ly + o + GSR_SSIM_R][lx + GSR_SSIM_R]);
        }
    }
    l1 = wave_sum_d(l1); ss = wave_sum_d(ss);
    if ((tid & 63) == 0) { s_red[tid >> 6][0] = l1; s_red[tid >> 6][1] = ss; }
    __syncthreads();
    if (tid < 2) {
        const double t = s_red[0][tid] + s_red[1][tid] + s_red[2][tid] + s_red[3][tid];
        if (t != 0.0) atomicAdd(&a.sums[tid], t);
    }
}

__global__ void __launch_bounds__(GSR_SSIM_THREADS) k_ssim_bwd(SsimArgs a)
{
    __shared__ __attribute__((aligned(16))) float s_m[3][GSR_SSIM_H][GSR_SSIM_S];
    __shared__ __attribute__((aligned(16))) float s_h[3][GSR_SSIM_H][GSR_SSIM_T];
    const int tid = threadIdx.x;
    const int ch = blockIdx.z;
    const int x0 = blockIdx.x * GSR_SSIM_T, y0 = blockIdx.y * GSR_SSIM_T;
    const size_t N = (size_t)a.W * a.H;
    for (int i = tid; i < GSR_SSIM_H * GSR_SSIM_H; i += GSR_SSIM_THREADS) {
        const int r = i / GSR_SSIM_H, c = i - r * GSR_SSIM_H;
        const int gx = x0 + c - GSR_SSIM_R, gy = y0 + r - GSR_SSIM_R;
        const bool in = gx >= 0 && gx < a.W && gy >= 0 && gy < a.H;          // no output pixel outside the image
        const size_t o = ch * N + (size_t)gy * a.W + gx;
#pragma unroll
        for (int m = 0; m < 3; m++) s_m[m][r][c] = in ? a.maps[3 * m * N + o] : 0.f;
    }
    __syncthreads();
#define GSR_SSIM_LOAD_BWD                                                                                                    \
        _Pragma("unroll") for (int q = 0; q < 3; q++) {                                                                      \
            _Pragma("unroll") for (int v = 0; v < 3; v++) {                                                                  \
                const float4 mv = *reinterpret_cast<const float4*>(&s_m[q][r][c0 + 4 * v]);                                 \
                in[q][4 * v] = mv.x; in[q][4 * v + 1] = mv.y; in[q][4 * v + 2] = mv.z; in[q][4 * v + 3] = mv.w;              \
            }                                                                                                                \
            const float2 mv = *reinterpret_cast<const float2*>(&s_m[q][r][c0 + 12]); in[q][12] = mv.x; in[q][13] = mv.y;     \
        }
#define GSR_SSIM_STORE3                                                                                                      \
        _Pragma("unroll") for (int q = 0; q < 3; q++)                                                                        \
            *reinterpret_cast<float4*>(&s_h[q][r][c0]) = make_float4(acc[q][0], acc[q][1], acc[q][2], acc[q][3]);
    GSR_SSIM_HPASS(3, GSR_SSIM_LOAD_BWD, GSR_SSIM_STORE3)
#undef GSR_SSIM_LOAD_BWD
#undef GSR_SSIM_STORE3
    __syncthreads();
    const int lx = tid & (GSR_SSIM_T - 1), ly = tid >> 5;
    float g[3][4];
#pragma unroll
    for (int q = 0; q < 3; q++) {
        float col[14];
#pragma unroll
        for (int j = 0; j < 14; j++) col[j] = s_h[q][4 * ly + j][lx];
#pragma unroll
        for (int o = 0; o < 4; o++) {
            float t = 0.f;
#pragma unroll
            for (int k = 0; k < 2 * GSR_SSIM_R + 1; k++) t += a.w[k] * col[o + k];
            g[q][o] = t;
        }
    }
    const int px = x0 + lx;
    const float inv3n = 1.f / (3.f * (float)N);
#pragma unroll
    for (int o = 0; o < 4; o++) {
        const int py = y0 + 4 * ly + o;
        if (px >= a.W || py >= a.H) continue;
        const size_t oo = ch * N + (size_t)py * a.W + px;
        const float x = a.img[oo], y = a.gt[oo];
        const float d = x - y;
        const float sgn = (d > 0.f) ? 1.f : ((d < 0.f) ? -1.f : 0.f);
        // loss = (1 - lambda) mean|x - y| + lambda (1 - mean ssim_map)
        a.dL_dimage[oo] = (1.f - a.lambda_dssim) * sgn * inv3n - a.lambda_dssim * inv3n * (g[0][o] + 2.f * x * g[1][o] + y * g[2][o]);
    }
}
#undef GSR_SSIM_HPASS

// Pseudo-depth term of train.py:96-108: w_d * min(1 - rho(-m, d), 1 - rho(1 / (m + 200), d)), rho = Pearson
// correlation over all pixels (torchmetrics pearson_corrcoef: cov / sqrt(var_x var_y), clamped to [-1, 1]).
struct PearsonArgs {
    int n;
    const float* depth; const float* pseudo;
    double* sums;         // [2..9]: sum d, sum dd, sum a, sum aa, sum ad, sum b, sum bb, sum bd   (a = -m, b = 1/(m+200))
    float weight;
    float* dL_ddepth;
    float* out;           // [0] loss, [1] Ll1, [2] ssim, [3] pseudo-depth loss
    float lambda_dssim; int npix3;      // for the final scalar
};
__global__ void __launch_bounds__(GSR_BLOCK) k_pearson_sums(PearsonArgs a)
{
    __shared__ double s_red[4][8];
    double v[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    for (int i = blockIdx.x * GSR_BLOCK + threadIdx.x; i < a.n; i += gridDim.x * GSR_BLOCK) {
        const double d = (double)a.depth[i], m = (double)a.pseudo[i];
        const double xa = -m, xb = (double)(1.0f / ((float)m + 200.f));
        v[0] += d; v[1] += d * d; v[2] += xa; v[3] += xa * xa; v[4] += xa * d; v[5] += xb; v[6] += xb * xb; v[7] += xb * d;
    }
#pragma unroll
    for (int q = 0; q < 8; q++) {
        const double t = wave_sum_d(v[q]);
        if ((threadIdx.x & 63) == 0) s_red[threadIdx.x >> 6][q] = t;
    }
    __syncthreads();
    if (threadIdx.x < 8) {
        const double t = s_red[0][threadIdx.x] + s_red[1][threadIdx.x] + s_red[2][threadIdx.x] + s_red[3][threadIdx.x];
        if (t != 0.0) atomicAdd(&a.sums[2 + threadIdx.x], t);
    }
}
// rho and the coefficients of d(1 - rho)/dd_i = -(x_i - mx) / (n sx sd) + rho (d_i - md) / (n sd^2)
__device__ __forceinline__ void pearson_terms(double n, double sx, double sxx, double sd, double sdd, double sxd, double& rho,
                                              double& mx, double& md, double& cx, double& cd)
{
    mx = sx / n; md = sd / n;
    const double vx = sxx / n - mx * mx, vd = sdd / n - md * md, cov = sxd / n - mx * md;
    const double den = sqrt(vx * vd);
    rho = cov / den;
    const bool clamped = rho > 1.0 || rho < -1.0;       // torch.clamp: no gradient through a clamped value
    rho = fmin(1.0, fmax(-1.0, rho));
    cx = clamped ? 0.0 : -1.0 / (n * den);
    cd = clamped ? 0.0 : rho / (n * vd);
}
__global__ void __launch_bounds__(GSR_BLOCK) k_train_loss_finish(PearsonArgs a, const double* ssim_sums)
{
    double rho_a = 0, rho_b = 0, mxa = 0, mxb = 0, md = 0, cxa = 0, cxb = 0, cda = 0, cdb = 0, md2 = 0;
    float pd = 0.f;
    bool use_a = true;
    if (a.depth != nullptr) {
        const double n = (double)a.n;
        const double* s = a.sums + 2;
        pearson_terms(n, s[2], s[3], s[0], s[1], s[4], rho_a, mxa, md, cxa, cda);
        pearson_terms(n, s[5], s[6], s[0], s[1], s[7], rho_b, mxb, md2, cxb, cdb);
        use_a = !((1.0 - rho_b) < (1.0 - rho_a));          // Python min(): the first argument wins ties
        pd = (float)(use_a ? 1.0 - rho_a : 1.0 - rho_b);
        for (int i = blockIdx.x * GSR_BLOCK + threadIdx.x; i < a.n; i += gridDim.x * GSR_BLOCK) {
            const double d = (double)a.depth[i], m = (double)a.pseudo[i];
            const double x = use_a ? -m : (double)(1.0f / ((float)m + 200.f));
            const double g = use_a ? cxa * (x - mxa) + cda * (d - md) : cxb * (x - mxb) + cdb * (d - md);
            a.dL_ddepth[i] = a.weight * (float)g;
        }
    }
    if (blockIdx.x == 0 && threadIdx.x == 0) {
        const float l1 = (float)(ssim_sums[0] / (double)a.npix3), ss = (float)(ssim_sums[1] / (double)a.npix3);
        a.out[1] = l1; a.out[2] = ss; a.out[3] = pd;
        a.out[0] = (1.0f - a.lambda_dssim) * l1 + a.lambda_dssim * (1.0f - ss) + ((a.depth != nullptr) ? a.weight * pd : 0.f);
    }
}

// Densification statistics of train.py:142-145 / gaussian_model.py:405-407 in one pass over the Gaussians.
__global__ void __launch_bounds__(GSR_BLOCK) k_densification_stats(int P, const int* radii, const float* dL_dmean2D,
                                                                   float* max_radii2D, float* xyz_gradient_accum, float* denom)
{
    const int i = blockIdx.x * GSR_BLOCK + threadIdx.x;
    if (i >= P) return;
    const int r = radii[i];
    if (r <= 0) return;                                              // visibility_filter = radii > 0
    max_radii2D[i] = fmaxf(max_radii2D[i], (float)r);
    const float gx = dL_dmean2D[3 * i], gy = dL_dmean2D[3 * i + 1];
    xyz_gradient_accum[i] += sqrtf(gx * gx + gy * gy);               // torch.norm(grad[:, :2], dim=-1)
    denom[i] += 1.f;
}

// ---------------------------------------------------------------------------------------------
// Map on-disk rows -> device layout.  Replaces the host-side column gathering of
// load_ply (gs_localization/pipelines/tools/gaussian_model.py:377-467, gaussian_splatting/scene/
// gaussian_model.py:215-256) and, for the read-only localisation map, the activation getters that the
// reference re-evaluates in every render() (tools/gaussian_model.py:77-96: exp, sigmoid, normalize, cat).
// Input: the P vertex rows exactly as stored in point_cloud.ply (row_floats f32 properties each), uploaded
// as they are.  One wave per 64 rows: the rows arrive as one coalesced stream into LDS, each lane then
// converts its own row.  HBM-bound byte work: 4*row_floats B in, (19 + 3M)*4 B out per Gaussian.
// ---------------------------------------------------------------------------------------------
#define GSR_PLY_MAX_REST 45
struct PlyCols {             // float index of each property inside a row
    int xyz[3], f_dc[3], f_rest[GSR_PLY_MAX_REST], opacity, scale[3], rot[4];
    int n_rest;              // 3 * ((D + 1)^2 - 1)
};
struct PlyMapArgs {
    int P, row_floats, activate, M;
    const float* rows;
    float* means3D; float* shs; float* opacities; float* scales; float* rotations;
    PlyCols c;
};
// RF / MM: compile-time row length and SH coefficient count (the index arithmetic is all divisions by them);
// 0 = take them from the arguments.
template <int RF, int MM>
__global__ void __launch_bounds__(64) k_map_from_ply_rows(PlyMapArgs a)
{
    const int rf = RF ? RF : a.row_floats, mm = RF ? MM : a.M;
    extern __shared__ float s_rows[];            // 64 rows, odd row stride (conflict-free column reads)
    __shared__ int s_col[3 * 16];                // source column of every element of one [M,3] feature row
    __shared__ float s_qn[64];                   // per row: 1 / max(|q|, eps)   (F.normalize, eps 1e-12)
    const int lane = threadIdx.x;
    const int base = blockIdx.x * 64;
    const int nrow = min(64, a.P - base);
    const int rs = rf | 1;
    const float* src = a.rows + (size_t)base * rf;
    // the block's rows are contiguous in the file: one coalesced stream, 16 B per lane when the buffer allows
    const int nfl = nrow * rf;
    if ((reinterpret_cast<uintptr_t>(src) & 15u) == 0) {
        const float4* src4 = reinterpret_cast<const float4*>(src);
        for (int i4 = lane; i4 < (nfl >> 2); i4 += 64) {
            const float4 v = src4[i4];
            const float vv[4] = {v.x, v.y, v.z, v.w};
            int r = (4 * i4) / rf, c = 4 * i4 - r * rf;
#pragma unroll
            for (int k = 0; k < 4; k++) {
                s_rows[r * rs + c] = vv[k];
                if (++c == rf) { c = 0; r++; }
            }
        }
        for (int i = (nfl & ~3) + lane; i < nfl; i += 64) {
            const int r = i / rf;
            s_rows[r * rs + (i - r * rf)] = src[i];
        }
    } else {
        for (int i = lane; i < nfl; i += 64) {
            const int r = i / rf;
            s_rows[r * rs + (i - r * rf)] = src[i];
        }
    }
    // features: [P, M, 3], coefficient-major, RGB innermost = cat(features_dc, features_rest) after the
    // reference's reshape (P, 3, M-1) + transpose(1, 2): f_rest_{c*(M-1)+k} is coefficient 1+k of channel c
    const int nr = mm - 1;
    if (lane < 3 * mm) {
        const int kk = lane / 3, c = lane - kk * 3;
        s_col[lane] = (kk == 0) ? a.c.f_dc[c] : a.c.f_rest[c * nr + (kk - 1)];
    }
    __syncthreads();
    if (lane < nrow) {
        const float* row = s_rows + lane * rs;
        const float q0 = row[a.c.rot[0]], q1 = row[a.c.rot[1]], q2 = row[a.c.rot[2]], q3 = row[a.c.rot[3]];
        s_qn[lane] = a.activate ? fmaxf(sqrtf(q0 * q0 + q1 * q1 + q2 * q2 + q3 * q3), 1e-12f) : 1.f;
        const float o = row[a.c.opacity];
        a.opacities[(size_t)base + lane] = a.activate ? 1.0f / (1.0f + expf(-o)) : o;          // torch.sigmoid
    }
    __syncthreads();
    // every output tensor's slice of this block is contiguous: consecutive lanes write consecutive floats
    const int w = 3 * mm;
    float* shs = a.shs + (size_t)base * w;
    if ((reinterpret_cast<uintptr_t>(shs) & 15u) == 0 && ((nrow * w) & 3) == 0) {
        for (int e4 = lane; e4 < (nrow * w) >> 2; e4 += 64) {
            int r = (4 * e4) / w, c = 4 * e4 - r * w;
            float vv[4];
#pragma unroll
            for (int k = 0; k < 4; k++) {
                vv[k] = s_rows[r * rs + s_col[c]];
                if (++c == w) { c = 0; r++; }
            }
            reinterpret_cast<float4*>(shs)[e4] = make_float4(vv[0], vv[1], vv[2], vv[3]);
        }
    } else {
        for (int e = lane; e < nrow * w; e += 64) {
            const int r = e / w;
            shs[e] = s_rows[r * rs + s_col[e - r * w]];
        }
    }
    float* means = a.means3D + (size_t)base * 3;
    float* scales = a.scales + (size_t)base * 3;
    for (int e = lane; e < nrow * 3; e += 64) {
        const int r = e / 3, c = e - r * 3;
        means[e] = s_rows[r * rs + a.c.xyz[c]];
        const float sv = s_rows[r * rs + a.c.scale[c]];
        scales[e] = a.activate ? expf(sv) : sv;                                                  // torch.exp
    }
    float* rots = a.rotations + (size_t)base * 4;
    for (int e = lane; e < nrow * 4; e += 64) {
        const int r = e >> 2, c = e & 3;
        rots[e] = s_rows[r * rs + a.c.rot[c]] / s_qn[r];
    }
}

// ---------------------------------------------------------------------------------------------
// Pose-refinement epilogue: the ~130 tiny launches the reference's Python loop
// issues per iteration for the tracking loss, its autograd backward, Adam and update_pose become two.
// ---------------------------------------------------------------------------------------------
// Tracking loss of gs_localization/pipelines/tools/descent_utils.py:85-123 and its gradient w.r.t. the
// rendered image / depth and the exposure pair (a, b):
//   image_ab = exp(a) image + b;  L = mean(om |image_ab gm - gt gm|) [+ w_d mean(|depth dm - gt_d dm|)]
//   om = opacity > thr, gm = grad_mask, dm = (gt_d > 0.01) om gm.   No gradient flows into opacity.
struct LossArgs {
    int W, H;
    const float* image; const float* depth; const float* opacity; const float* gt_image; const float* gt_depth;
    const uint8_t* grad_mask; const float* exposure; float opacity_thr, depth_w; int monocular;
    float* dL_dimage; float* dL_ddepth; float* dL_dalpha; float* out;     // out[0]=loss, [1]=dL/da, [2]=dL/db
    // native loop (nullable): per-superblock words that this iteration's forward has consumed and the next one
    // starts from zero -- cleared here instead of by two memsets per iteration
    uint32_t* clear_a; float* clear_b; int clear_n;
    LoopGuard guard;
};
__global__ void __launch_bounds__(GSR_BLOCK) k_tracking_loss(LossArgs a)
{
    __shared__ float s_red[4][3];
    if (a.guard.frozen()) return;
    if (blockIdx.x == 0 && a.clear_b != nullptr)
        for (int i = threadIdx.x; i < a.clear_n; i += GSR_BLOCK) { if (a.clear_a != nullptr) a.clear_a[i] = 0u; a.clear_b[i] = 0.f; }
    const int n = a.W * a.H;
    const float ea = expf(a.exposure[0]), eb = a.exposure[1];
    const float inv3n = 1.f / (3.f * (float)n), invn = 1.f / (float)n;
    float l = 0.f, da = 0.f, db = 0.f;
    // grid-stride: few blocks, so that the three result words see few same-address atomics
    for (int i = blockIdx.x * GSR_BLOCK + threadIdx.x; i < n; i += gridDim.x * GSR_BLOCK) {
        const bool om = a.opacity[i] > a.opacity_thr;
        const float gm = a.grad_mask[i] ? 1.f : 0.f;
        const float w = om ? gm : 0.f;
#pragma unroll
        for (int c = 0; c < 3; c++) {
            const float img = a.image[(size_t)c * n + i];
            const float d = (ea * img + eb) * gm - a.gt_image[(size_t)c * n + i] * gm;
            if (om) l += fabsf(d) * inv3n;
            const float g = w * sgnf(d) * inv3n;
            a.dL_dimage[(size_t)c * n + i] = g * ea;
            da += g * ea * img;
            db += g;
        }
        float gdp = 0.f;
        if (!a.monocular) {
            const float gd = a.gt_depth[i];
            const float dm = (gd > 0.01f && om) ? gm : 0.f;
            const float dd = a.depth[i] * dm - gd * dm;
            l += a.depth_w * fabsf(dd) * invn;
            gdp = a.depth_w * dm * sgnf(dd) * invn;
        }
        a.dL_ddepth[i] = gdp;
        a.dL_dalpha[i] = 0.f;
    }
    l = wave_sum(l); da = wave_sum(da); db = wave_sum(db);
    const int wv = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0) { s_red[wv][0] = l; s_red[wv][1] = da; s_red[wv][2] = db; }
    __syncthreads();
    if (threadIdx.x < 3) {
        const float t = s_red[0][threadIdx.x] + s_red[1][threadIdx.x] + s_red[2][threadIdx.x] + s_red[3][threadIdx.x];
        if (t != 0.f) atomicAdd(&a.out[threadIdx.x], t);
    }
}

// K10  near-plane visibility (replaces rasterizer_impl.cu:54-66 checkFrustum)
__global__ void __launch_bounds__(GSR_BLOCK) k_mark_visible(int P, const float* means, const float* view, uint8_t* present)
{
    const int idx = blockIdx.x * GSR_BLOCK + threadIdx.x;
    if (idx >= P) return;
    const float3 p = make_float3(means[3 * idx], means[3 * idx + 1], means[3 * idx + 2]);
    present[idx] = xform4x3(p, view).z > 0.2f ? 1 : 0;
}

// bench-only statistics: V, R under the reference's bounding rule, instances binned, R_eff
__global__ void __launch_bounds__(GSR_BLOCK) k_stats_gauss(int P, const int* radii, const ushort4* rects, unsigned long long* out)
{
    const int idx = blockIdx.x * GSR_BLOCK + threadIdx.x;
    unsigned long long v = 0, r = 0;
    if (idx < P && radii[idx] > 0) {
        v = 1;
        const ushort4 rc = rects[idx];
        r = (unsigned long long)(rc.z - rc.x) * (rc.w - rc.y);      // the reference's bounding-square count
    }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) { v += __shfl_xor(v, off, 64); r += __shfl_xor(r, off, 64); }
    if ((threadIdx.x & 63) == 0) { atomicAdd(&out[0], v); atomicAdd(&out[1], r); }
}
__global__ void __launch_bounds__(GSR_BLOCK) k_stats_tiles(int W, int H, int gx, const uint32_t* n_contrib, const uint2* ranges,
                                                           unsigned long long* out)
{
    if (threadIdx.x == 0) { const uint2 rg = ranges[blockIdx.x]; atomicAdd(&out[3], (unsigned long long)(rg.y - rg.x)); }
    __shared__ int wm[4];
    const int tx = blockIdx.x % gx, ty = blockIdx.x / gx;
    const int px = tx * GSR_TILE + (threadIdx.x & 15), py = ty * GSR_TILE + (threadIdx.x >> 4);
    int m = (px < W && py < H) ? (int)n_contrib[W * py + px] : 0;
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) m = max(m, __shfl_xor(m, off, 64));
    if ((threadIdx.x & 63) == 0) wm[threadIdx.x >> 6] = m;
    __syncthreads();
    if (threadIdx.x == 0) atomicAdd(&out[2], (unsigned long long)max(max(wm[0], wm[1]), max(wm[2], wm[3])));
}

}  // namespace gsr
