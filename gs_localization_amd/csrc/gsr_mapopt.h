// gsr_mapopt.h -- the optimiser step of a Gaussian map and the pruning that goes with it: what gaussian_splatting/train.py:155-157 leaves
// to torch (Adam over six tensors, ~12 launches each; the rewriting of its state at every prune, scene/gaussian_model.py:269-300).
//
//   k_grad_norm, k_grad_norm_finish   the 2-norm over many tensors and the coefficient that clips it, on the device
//   k_adamw                           p, m, v of many tensors in one launch, moments in 32 bits
//   k_adamw8                          the same with a byte for each moment
//   k_moments8                        the values those bytes stand for
//   k_evict_*                         accumulated compositing weights -> the rows that stay -> every tensor compacted
//
// Arithmetic: 32 bits, every operation rounded by itself (the build contracts nothing), so the results are those of the same sequence
// of elementwise torch operations, bit for bit; the step's scalars and all long sums are held in 64 bits and rounded once.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace gsr {

#define GSR_OPT_MAX 40          // tensors of one launch: their table travels as a kernel argument (at most 4 KB), nothing is uploaded
#define GSR_OPT_CHUNK 4096      // elements a workgroup takes at a time: 16 per lane
#define GSR_OPT_THREADS 256
#define GSR_OPT_WINDOW 256      // elements that share a window of the 8-bit root: four per lane of a wave
#define GSR_NORM_MAX 160

enum { GSR_T_F32 = 0, GSR_T_BF16 = 1, GSR_T_F16 = 2, GSR_T_ALIGNED = 256 };          // aligned: opt_load4 may be used

__device__ __forceinline__ float opt_load(const void* p, long long i, int type)
{
    if (type == GSR_T_F32) return static_cast<const float*>(p)[i];
    if (type == GSR_T_BF16) return __uint_as_float((uint32_t)static_cast<const uint16_t*>(p)[i] << 16);
    return (float)static_cast<const _Float16*>(p)[i];
}
// half precision: rounded to nearest even, once, from the 32-bit result (no stochastic rounding: what an update smaller than half a
// step does to a half-precision parameter is nothing, as with torch)
__device__ __forceinline__ void opt_store(void* p, long long i, int type, float x)
{
    if (type == GSR_T_F32) static_cast<float*>(p)[i] = x;
    else if (type == GSR_T_BF16) static_cast<__bf16*>(p)[i] = (__bf16)x;
    else static_cast<_Float16*>(p)[i] = (_Float16)x;
}

// Four elements at once, i a multiple of four, the pointer aligned to four of them (16 bytes in 32 bits, 8 in half precision).
typedef float opt_f4 __attribute__((ext_vector_type(4)));
typedef uint32_t opt_u2 __attribute__((ext_vector_type(2)));
typedef __bf16 opt_b4 __attribute__((ext_vector_type(4)));
typedef _Float16 opt_h4 __attribute__((ext_vector_type(4)));
// STREAM: past the caches (non-temporal), for a launch whose data do not fit the 256 MB behind the L2 anyway: without it the lines
// that a step leaves there only push out one another.  The rule is opt_stream() (gsr_mapopt_api.h), with both sides measured.
template <bool STREAM, class T> __device__ __forceinline__ T opt_get(const T* p) { return STREAM ? __builtin_nontemporal_load(p) : *p; }
template <bool STREAM, class T> __device__ __forceinline__ void opt_put(T* p, T x) { if (STREAM) __builtin_nontemporal_store(x, p); else *p = x; }
template <int TYPE, bool STREAM>
__device__ __forceinline__ opt_f4 opt_load4(const void* p, long long i)
{
    if (TYPE == GSR_T_F32) return opt_get<STREAM>(reinterpret_cast<const opt_f4*>(static_cast<const float*>(p) + i));
    const opt_u2 x = opt_get<STREAM>(reinterpret_cast<const opt_u2*>(static_cast<const uint16_t*>(p) + i));
    if (TYPE == GSR_T_F16) return __builtin_convertvector(__builtin_bit_cast(opt_h4, x), opt_f4);
    opt_f4 r;
    r.x = __uint_as_float(x.x << 16); r.y = __uint_as_float(x.x & 0xffff0000u); r.z = __uint_as_float(x.y << 16); r.w = __uint_as_float(x.y & 0xffff0000u);
    return r;
}
template <int TYPE, bool STREAM>
__device__ __forceinline__ void opt_store4(void* p, long long i, opt_f4 x)
{
    if (TYPE == GSR_T_F32) { opt_put<STREAM>(reinterpret_cast<opt_f4*>(static_cast<float*>(p) + i), x); return; }
    const opt_u2 h = TYPE == GSR_T_F16 ? __builtin_bit_cast(opt_u2, __builtin_convertvector(x, opt_h4)) : __builtin_bit_cast(opt_u2, __builtin_convertvector(x, opt_b4));
    opt_put<STREAM>(reinterpret_cast<opt_u2*>(static_cast<uint16_t*>(p) + i), h);
}
template <int TYPE> __device__ __forceinline__ float opt_load1(const void* p, long long i) { return opt_load(p, i, TYPE); }

// ---- the norm of the gradients --------------------------------------------------------------------------------------------------

struct NormTensor { const void* g; long long n; uint32_t first; int type; };          // first: its first chunk in the launch; type | GSR_T_ALIGNED
struct NormArgs {
    int count;
    uint32_t chunks;
    double* partial;            // one sum per workgroup
    float max_norm; float* out; // out: nullable; a launch of one workgroup that writes the result itself
    NormTensor t[GSR_NORM_MAX];
};

template <class T>
__device__ __forceinline__ int opt_find(const T* t, int count, uint32_t chunk)          // the last tensor that starts at or before `chunk`
{
    int lo = 0, hi = count - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (t[mid].first <= chunk) lo = mid; else hi = mid - 1;
    }
    return lo;
}

__device__ __forceinline__ double opt_block_sum(double x, double* s)          // total over the workgroup's four waves, in thread 0
{
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) x += __shfl_xor(x, off, 64);
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = x;
    __syncthreads();
    return threadIdx.x == 0 ? ((s[0] + s[1]) + (s[2] + s[3])) : 0.0;
}

// A product of two floats is exact in a double: one rounding per element, 2^-53 of the running sum.
__device__ __forceinline__ void norm_add(double& sum, float x) { sum = __builtin_fma((double)x, (double)x, sum); }

template <int TYPE>
__device__ __forceinline__ void norm_chunk(const NormTensor& t, long long base, double (&sum)[4])
{
    if (t.type & GSR_T_ALIGNED) {
        opt_f4 x[4];
#pragma unroll
        for (int u = 0; u < 4; u++) {
            const long long i = base + 4 * (u * GSR_OPT_THREADS + (int)threadIdx.x);
            x[u] = 0.0f;
            if (i + 4 <= t.n) x[u] = opt_load4<TYPE, false>(t.g, i);
            else if (i < t.n) { x[u].x = opt_load1<TYPE>(t.g, i); if (i + 1 < t.n) x[u].y = opt_load1<TYPE>(t.g, i + 1); if (i + 2 < t.n) x[u].z = opt_load1<TYPE>(t.g, i + 2); }
        }
#pragma unroll
        for (int u = 0; u < 4; u++) { norm_add(sum[0], x[u].x); norm_add(sum[1], x[u].y); norm_add(sum[2], x[u].z); norm_add(sum[3], x[u].w); }
    } else {
        for (int k = threadIdx.x; k < GSR_OPT_CHUNK && base + k < t.n; k += GSR_OPT_THREADS) norm_add(sum[0], opt_load1<TYPE>(t.g, base + k));
    }
}

// torch.nn.utils.clip_grad_norm_'s coefficient: min(1, max_norm / (norm + 1e-6)), a NaN norm stays one.
__device__ __forceinline__ void norm_out(double sum, float max_norm, float* out)
{
    const float norm = (float)sqrt(sum);
    const float c = max_norm / (norm + 1e-6f);
    out[0] = norm;
    out[1] = c > 1.0f ? 1.0f : c;
}

__global__ void __launch_bounds__(GSR_OPT_THREADS) k_grad_norm(NormArgs a)
{
    __shared__ double s[4];
    double sum[4] = {0.0, 0.0, 0.0, 0.0};
    for (uint32_t c = blockIdx.x; c < a.chunks; c += gridDim.x) {
        const NormTensor& t = a.t[opt_find(a.t, a.count, c)];
        const long long base = (long long)(c - t.first) * GSR_OPT_CHUNK;
        const int type = t.type & 15;
        if (type == GSR_T_F32) norm_chunk<GSR_T_F32>(t, base, sum);
        else if (type == GSR_T_BF16) norm_chunk<GSR_T_BF16>(t, base, sum);
        else norm_chunk<GSR_T_F16>(t, base, sum);
    }
    const double total = opt_block_sum((sum[0] + sum[1]) + (sum[2] + sum[3]), s);
    if (threadIdx.x == 0) { if (a.out) norm_out(total, a.max_norm, a.out); else a.partial[blockIdx.x] = total; }
}

// The partial sums in a fixed order: the result does not depend on which workgroup ran when.
__global__ void __launch_bounds__(GSR_OPT_THREADS) k_grad_norm_finish(const double* __restrict__ partial, int n, float max_norm, float* __restrict__ out)
{
    __shared__ double s[4];
    double sum = 0.0;
    for (int i = threadIdx.x; i < n; i += GSR_OPT_THREADS) sum += partial[i];
    sum = opt_block_sum(sum, s);
    if (threadIdx.x == 0) norm_out(sum, max_norm, out);
}

// ---- AdamW ----------------------------------------------------------------------------------------------------------------------

struct OptTensor {
    void* p; const void* g;
    void* s0;                   // 32 bits: exp_avg; 8 bits: codes of the root
    void* s1;                   // 32 bits: exp_avg_sq; 8 bits: codes of the ratio
    uint8_t* window;            // 8 bits: one byte per GSR_OPT_WINDOW elements
    double* clock;              // beta1^t, beta2^t, t, (word of the last workgroup's ticket)
    const double* lr_device;    // nullable: a rate that a replayed graph reads anew
    double lr, decay;
    long long n;
    uint32_t first;             // its first workgroup in the launch
    uint32_t key;               // 8 bits: seed and place
    int types;                  // parameter | gradient << 4 | GSR_T_ALIGNED
    float unit;                 // 8 bits: the step of the ratios that it comes with (of the betas they were stored with)
};
struct OptArgs {
    int count;
    double beta1, beta2;
    float b1, b2, c1, c2, eps;  // (c = 1 - beta)
    float per_unit;             // 8 bits: steps of the ratio per one, as this step stores it
    const float* clip;          // nullable: (norm, coefficient)
    OptTensor t[GSR_OPT_MAX];
};

__device__ __forceinline__ bool opt_aligned4(const void* p) { return ((uintptr_t)p & 3) == 0; }
__device__ __forceinline__ float opt_uniform(float x) { return __uint_as_float(__builtin_amdgcn_readfirstlane((int)__float_as_uint(x))); }
// The step's scalars, formed in 64 bits: by every wave, behind the loads of its first elements (two divisions and a root of 64 bits
// under their latency), kept in scalar registers.
//
// The step counts live on the device, so that a captured graph goes on counting.  They may advance once every workgroup has read them.  A
// launch of up to GSR_OPT_TICKETS workgroups does it by itself: a workgroup draws a ticket when it is done (the fourth word of the
// launch's first clock, zero between launches), and the one that drew the last advances the clocks.  No fence: nothing but "has read" is
// handed over, and what a wave has stored it has computed from the clock (a release at device scope writes the XCD's L2 back, 57 ns
// per workgroup).  Same-address atomics take turns, so a larger launch leaves it to k_adamw_advance behind it: 34.5 M
// elements, 8424 workgroups: 302 us with tickets and fences, 209 with tickets, 167 + 4 with the launch.  A tensor stepped again and again, with
// tickets / with the launch: 256 workgroups 9.4 / 11.1 us, 384 11.4 / 11.1, 512 13.5 / 11.3, 768 37 / 16, 1024 62 / 20 (8 bits 10.2 / 11.4,
// 12.0 / 11.5, 13.9 / 11.5, 17.8 / 13.7, 21.6 / 17.7): 512 is not far above the border.
#define GSR_OPT_TICKETS 512
struct OptRates { float shrink, rate, unbias; uint32_t key; };
__device__ __forceinline__ OptRates opt_rates(const OptArgs& a, const OptTensor& t)
{
    const double lr = t.lr_device ? *t.lr_device : t.lr;
    const double b1t = t.clock[0] * a.beta1, b2t = t.clock[1] * a.beta2;
    OptRates r;
    r.shrink = opt_uniform((float)(1.0 - lr * t.decay));
    r.rate = opt_uniform((float)((1.0 / (1.0 - b1t)) * lr));
    r.unbias = opt_uniform((float)(1.0 / sqrt(1.0 - b2t)));
    r.key = (uint32_t)__builtin_amdgcn_readfirstlane((int)(t.key + (uint32_t)(t.clock[2] + 1.0)));
    return r;
}
__device__ __forceinline__ void opt_advance(const OptArgs& a)          // one wave
{
    for (int i = threadIdx.x; i < a.count; i += 64) {
        double* c = a.t[i].clock;
        c[0] *= a.beta1; c[1] *= a.beta2; c[2] += 1.0;
        if (i == 0) c[3] = 0.0;
    }
}
__device__ __forceinline__ void opt_end(const OptArgs& a)          // every wave of the workgroup
{
    if (gridDim.x > GSR_OPT_TICKETS) return;
    __syncthreads();
    if (threadIdx.x >= 64) return;
    uint32_t ticket = 0;
    if (threadIdx.x == 0) ticket = __hip_atomic_fetch_add(reinterpret_cast<unsigned*>(a.t[0].clock + 3), 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    if ((uint32_t)__builtin_amdgcn_readfirstlane((int)ticket) == gridDim.x - 1u) opt_advance(a);
}
__global__ void __launch_bounds__(64) k_adamw_advance(OptArgs a) { opt_advance(a); }

__device__ __forceinline__ float adamw_one(const OptArgs& a, const OptRates& r, float coef, float p, float g, float& m, float& v)
{
    g *= coef;
    m = m * a.b1 + g * a.c1;
    v = v * a.b2 + (g * g) * a.c2;
    return p * r.shrink - (m / (sqrtf(v) * r.unbias + a.eps)) * r.rate;
}

template <int PT, int GT, bool STREAM>
__device__ __forceinline__ void adamw_chunk(const OptArgs& a, const OptTensor& t, float coef, long long base)
{
    float* pm = static_cast<float*>(t.s0);
    float* pv = static_cast<float*>(t.s1);
    opt_f4 p[4], g[4], m[4], v[4];
#pragma unroll
    for (int u = 0; u < 4; u++) {
        const long long i = base + 4 * (u * GSR_OPT_THREADS + (int)threadIdx.x);
        if (i + 4 <= t.n) {
            p[u] = opt_load4<PT, STREAM>(t.p, i); g[u] = opt_load4<GT, STREAM>(t.g, i);
            m[u] = opt_load4<GSR_T_F32, STREAM>(pm, i); v[u] = opt_load4<GSR_T_F32, STREAM>(pv, i);
        }
    }
    const OptRates r = opt_rates(a, t);
#pragma unroll
    for (int u = 0; u < 4; u++) {
        const long long i = base + 4 * (u * GSR_OPT_THREADS + (int)threadIdx.x);
        if (i + 4 <= t.n) {
#pragma unroll
            for (int k = 0; k < 4; k++) {
                float mm = m[u][k], vv = v[u][k];
                p[u][k] = adamw_one(a, r, coef, p[u][k], g[u][k], mm, vv);
                m[u][k] = mm; v[u][k] = vv;
            }
            opt_store4<PT, STREAM>(t.p, i, p[u]); opt_store4<GSR_T_F32, STREAM>(pm, i, m[u]); opt_store4<GSR_T_F32, STREAM>(pv, i, v[u]);
        } else {
            for (long long j = i; j < t.n; j++) opt_store(t.p, j, PT, adamw_one(a, r, coef, opt_load(t.p, j, PT), opt_load(t.g, j, GT), pm[j], pv[j]));
        }
    }
}

// Pointers that are not aligned to four elements: one element per lane and load, any types (34.5 M elements in f32: 294 us for 162).
__device__ __forceinline__ void adamw_chunk_unaligned(const OptArgs& a, const OptTensor& t, float coef, long long base)
{
    float* pm = static_cast<float*>(t.s0);
    float* pv = static_cast<float*>(t.s1);
    const int pt = t.types & 15, gt = (t.types >> 4) & 15;
    const OptRates r = opt_rates(a, t);
    for (int k = threadIdx.x; k < GSR_OPT_CHUNK && base + k < t.n; k += GSR_OPT_THREADS) {
        const long long j = base + k;
        opt_store(t.p, j, pt, adamw_one(a, r, coef, opt_load(t.p, j, pt), opt_load(t.g, j, gt), pm[j], pv[j]));
    }
}

template <bool STREAM>
__global__ void __launch_bounds__(GSR_OPT_THREADS) k_adamw(OptArgs a)
{
    const float coef = a.clip ? a.clip[1] : 1.0f;
    const OptTensor& t = a.t[opt_find(a.t, a.count, blockIdx.x)];          // (of no elements at all: a launch of one workgroup that advances the clocks)
    const long long base = (long long)(blockIdx.x - t.first) * GSR_OPT_CHUNK;
    switch (t.types) {
#define GSR_OPT_CASE(P, G) case P | G << 4 | GSR_T_ALIGNED: adamw_chunk<P, G, STREAM>(a, t, coef, base); break;
    GSR_OPT_CASE(0, 0) GSR_OPT_CASE(0, 1) GSR_OPT_CASE(0, 2) GSR_OPT_CASE(1, 0) GSR_OPT_CASE(1, 1) GSR_OPT_CASE(1, 2) GSR_OPT_CASE(2, 0) GSR_OPT_CASE(2, 1) GSR_OPT_CASE(2, 2)
#undef GSR_OPT_CASE
    default: adamw_chunk_unaligned(a, t, coef, base);
    }
    opt_end(a);
}

// ---- AdamW with a byte for each moment -------------------------------------------------------------------------------------------
//
// Stored are u = sqrt(v) and r = m / u.
//   u   the upper 13 bits of the float (sign, exponent, four bits of mantissa), minus 16 w + 1, in a byte; w, one byte per 256 elements,
//       places the window: sixteen binades under the block's largest root.  0 stands for 0; what is positive but lies under the window is
//       raised to code 1 (by a step, whose ratio is formed over the raised root, a smaller update, never a larger one; for an
//       eviction see evict_bytes).  Rounding is stochastic (19 random bits added under the kept ones: each rounding
//       exactly unbiased inside a binade): with beta2 = 0.999 the moment moves by 0.1 % per step, and rounded to the nearest sixteenth it
//       would stand still wherever it once was.
//   r   |m| <= B sqrt(v) whatever the gradients were, B = (1 - b1) / sqrt((1 - b2)(1 - b1^2 / b2)) (Cauchy-Schwarz over the two
//       exponential sums; 7.27 for 0.9 / 0.999): 127 steps of B / 127 to either side, stochastic (13 bits).  A momentum quantised for
//       itself could meet a root that its own block has rounded to almost nothing, and with train.py's eps = 1e-15 the quotient would
//       throw the splat across the scene; the ratio is the update, and cannot.  (B is that of the step which stores it; where a schedule
//       changes the betas, a momentum past it is stored as B.)
// The parameter is stepped with the moments before they are rounded.

__device__ __forceinline__ uint32_t opt_mix(uint32_t x)          // two rounds of xor-shift and odd multiplier (a bijection of 32 bits)
{
    x = (x ^ (x >> 16)) * 0x6C8E9CF5u;
    x = (x ^ (x >> 15)) * 0x2F7A5D1Bu;
    return x ^ (x >> 16);
}
__device__ __forceinline__ uint32_t opt_dither(uint32_t h, int k)          // the random bits of element 4 j + k from its quad's h: 19 | 13
{
    const uint32_t odd = k == 0 ? 0x00000001u : k == 1 ? 0xB5297A4Du : k == 2 ? 0x68E31DA5u : 0x1B56C4E9u;
    const uint32_t r = h * odd;
    return r ^ (r >> 15);
}
__device__ __forceinline__ float opt_decode(uint32_t code, uint32_t base)
{
    return code ? __uint_as_float((code + base) << 19) : 0.0f;
}
__device__ __forceinline__ uint32_t wave_max_u32(uint32_t v)          // over 64 lanes, in every lane (DPP, as wave_sum)
{
#define GSR_DPP_MAX(ctrl, rm) { const uint32_t o = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, ctrl, rm, 0xf, true); v = o > v ? o : v; }
    GSR_DPP_MAX(0x111, 0xf) GSR_DPP_MAX(0x112, 0xf) GSR_DPP_MAX(0x114, 0xf) GSR_DPP_MAX(0x118, 0xf) GSR_DPP_MAX(0x142, 0xa) GSR_DPP_MAX(0x143, 0xc)
#undef GSR_DPP_MAX
    return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}
__device__ __forceinline__ uint32_t opt_window(uint32_t largest)          // of the block's largest finite root, by its bits
{
    const int w = (int)(largest >> 23) - 15;          // its binade is the last but one: rounding up may need the next one's first value
    return w > 0 ? (uint32_t)w : 0u;
}

// sqrt of four values >= 0 (or infinite, or NaN), correctly rounded.  The instruction is within one ulp; s - ulp is nearer exactly if
// x <= s (s - ulp) (the midpoint's square is that plus ulp^2 / 4), s + ulp exactly if x > s (s + ulp).  sqrtf spends five more
// instructions on scaling arguments whose residual could underflow: here one test per wave sends those to it.
__device__ __forceinline__ void opt_sqrt4(const float (&x)[4], float (&s)[4])
{
    uint32_t least = __float_as_uint(x[0]) - 1u;          // (0 wraps to the largest: it needs no scaling)
#pragma unroll
    for (int k = 1; k < 4; k++) { const uint32_t b = __float_as_uint(x[k]) - 1u; least = b < least ? b : least; }
    if (__any(least < 0x0f800000u)) {          // something in (0, 2^-96]
#pragma unroll
        for (int k = 0; k < 4; k++) s[k] = sqrtf(x[k]);
        return;
    }
#pragma unroll
    for (int k = 0; k < 4; k++) {
        const float y = __builtin_amdgcn_sqrtf(x[k]);
        const float lo = __uint_as_float(__float_as_uint(y) - 1u), hi = __uint_as_float(__float_as_uint(y) + 1u);
        const float rl = __builtin_fmaf(-lo, y, x[k]), rh = __builtin_fmaf(-hi, y, x[k]);          // (at 0, infinity and NaN: NaN or 0, y stays)
        s[k] = rh > 0.0f ? hi : (rl <= 0.0f ? lo : y);
    }
}

// a / b for b in [2^-100, 2^100], by a refined reciprocal and one residual (Markstein's scheme: the quotient is the correctly rounded one but
// for residuals that underflow, of |a| under 2^-100).  The division operator spends five more instructions on scaling for any b; roots are
// in [2^-75, 2^64] here, squares of floats having been under them.
__device__ __forceinline__ float opt_div(float a, float b)
{
    float r = __builtin_amdgcn_rcpf(b);
    r = __builtin_fmaf(__builtin_fmaf(-b, r, 1.0f), r, r);
    const float q = a * r;
    return __builtin_fmaf(__builtin_fmaf(-b, q, a), r, q);
}

// One wave, NB blocks of 256 from `start`, four consecutive elements per lane, all loads in flight together.  FULL: every block lies inside the
// tensor and all pointers are aligned (PT, GT: the types), four blocks (two: 143 us for 132 over 47 M elements); otherwise element by
// element, any types, one block (four need 195 registers, which the whole kernel then has: 162 us for 128).
template <int PT, int GT, bool FULL, bool STREAM, int NB>
__device__ __forceinline__ void adamw8_blocks(const OptArgs& a, const OptTensor& t, float coef, long long start)
{
    const int pt = FULL ? PT : t.types & 15, gt = FULL ? GT : (t.types >> 4) & 15;
    const int lane = threadIdx.x & 63;
    uint8_t* rms = static_cast<uint8_t*>(t.s0);
    int8_t* ratio = static_cast<int8_t*>(t.s1);
    opt_f4 p[NB], g[NB];
    uint32_t cu[NB], cr[NB], old[NB];
#pragma unroll
    for (int b = 0; b < NB; b++) {
        const long long s = start + b * GSR_OPT_WINDOW, i = s + 4 * lane;
        p[b] = 0.0f; g[b] = 0.0f; cu[b] = cr[b] = old[b] = 0u;
        if (FULL) {
            p[b] = opt_load4<PT, STREAM>(t.p, i); g[b] = opt_load4<GT, STREAM>(t.g, i);
            cu[b] = opt_get<STREAM>(reinterpret_cast<const uint32_t*>(rms + i)); cr[b] = opt_get<STREAM>(reinterpret_cast<const uint32_t*>(ratio + i));
            old[b] = t.window[s / GSR_OPT_WINDOW];
        } else if (s < t.n) {
            old[b] = t.window[s / GSR_OPT_WINDOW];
#pragma unroll
            for (int k = 0; k < 4; k++)
                if (i + k < t.n) {
                    p[b][k] = opt_load(t.p, i + k, pt); g[b][k] = opt_load(t.g, i + k, gt);
                    cu[b] |= (uint32_t)rms[i + k] << (8 * k); cr[b] |= (uint32_t)(uint8_t)ratio[i + k] << (8 * k);
                }
        }
    }
    const OptRates r = opt_rates(a, t);
    const uint32_t key = opt_mix(r.key), lane_mul = (uint32_t)lane * 0x9E3779B1u;
#pragma unroll
    for (int b = 0; b < NB; b++) {
        const long long s = start + b * GSR_OPT_WINDOW, i = s + 4 * lane;
        if (!FULL && s >= t.n) break;          // (the whole wave)
        const uint32_t was = 16u * old[b] + 1u;
        float m1[4], v1[4], u1[4];
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const float u = opt_decode((cu[b] >> (8 * k)) & 255u, was);
            const float x = g[b][k] * coef;
            m1[k] = (((float)(int8_t)(cr[b] >> (8 * k)) * t.unit) * u) * a.b1 + x * a.c1;
            v1[k] = (u * u) * a.b2 + (x * x) * a.c2;
        }
        opt_sqrt4(v1, u1);
        uint32_t top = 0;
#pragma unroll
        for (int k = 0; k < 4; k++) top = __float_as_uint(u1[k]) > top ? __float_as_uint(u1[k]) : top;
        top = wave_max_u32(top);
        // An infinite root or a NaN (the whole wave, or none), roots of 0 over next to nothing, a divisor past opt_div's range.
        const bool rare = top >= 0x7f800000u || a.eps < 0x1p-100f || a.eps > 0x1p99f;
        if (rare) {
            top = 0;
#pragma unroll
            for (int k = 0; k < 4; k++) {
                p[b][k] = p[b][k] * r.shrink - (m1[k] / (u1[k] * r.unbias + a.eps)) * r.rate;
                if (__float_as_uint(u1[k]) >= 0x7f800000u) u1[k] = __builtin_inff();          // -> code 255; its neighbours' window is that of the finite ones
                else top = __float_as_uint(u1[k]) > top ? __float_as_uint(u1[k]) : top;
                if (m1[k] != m1[k]) m1[k] = 0.0f;
            }
            top = wave_max_u32(top);
        } else {
#pragma unroll
            for (int k = 0; k < 4; k++) p[b][k] = p[b][k] * r.shrink - opt_div(m1[k], u1[k] * r.unbias + a.eps) * r.rate;
        }
        const uint32_t w = opt_window(top), now = 16u * w + 1u;
        // (the upper half of the quad's number is the whole block's)
        const uint32_t h = opt_mix((((uint32_t)(s >> 2) * 0x9E3779B1u + lane_mul) ^ key) + (uint32_t)(s >> 34) * 0x85EBCA77u);
        uint32_t nu = 0, nr = 0;
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const uint32_t d = opt_dither(h, k), bits = __float_as_uint(u1[k]);
            int code = (int)((bits + (d >> 13)) >> 19) - (int)now;
            code = code < 1 ? 1 : (code > 255 ? 255 : code);
            code = bits == 0u ? 0 : code;
            const float u = __uint_as_float(((uint32_t)code + now) << 19);          // (of a code 0: some number, the quotient is not used)
            // An overflowed root's momentum may be infinite, or too large for opt_div over what code 255 stands for (2^-111 in a block of nothing else).
            const float over = rare ? m1[k] / u : opt_div(m1[k], u);
            // (the random bits times 2^-13 are exact: one rounding, as of a sum)
            float q = floorf(__builtin_fmaf((float)(d & 8191u), 1.0f / 8192.0f, over * a.per_unit));
            q = bits == 0u ? 0.0f : __builtin_amdgcn_fmed3f(q, -127.0f, 127.0f);
            nu |= (uint32_t)code << (8 * k);
            nr = __builtin_amdgcn_cvt_pk_u8_f32(q + 128.0f, k, nr);          // a whole number in 1 ... 255 into byte k
        }
        nr ^= 0x80808080u;          // less 128: two's complement
        if (FULL) {
            opt_store4<PT, STREAM>(t.p, i, p[b]);
            opt_put<STREAM>(reinterpret_cast<uint32_t*>(rms + i), nu); opt_put<STREAM>(reinterpret_cast<uint32_t*>(ratio + i), nr);
        } else {
#pragma unroll
            for (int k = 0; k < 4; k++)
                if (i + k < t.n) { opt_store(t.p, i + k, pt, p[b][k]); rms[i + k] = (uint8_t)(nu >> (8 * k)); ratio[i + k] = (int8_t)(nr >> (8 * k)); }
        }
        if (lane == 0) t.window[s / GSR_OPT_WINDOW] = (uint8_t)w;
    }
}

template <bool STREAM>
__global__ void __launch_bounds__(GSR_OPT_THREADS) k_adamw8(OptArgs a)
{
    const float coef = a.clip ? a.clip[1] : 1.0f;
    const OptTensor& t = a.t[opt_find(a.t, a.count, blockIdx.x)];
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const long long start = (long long)(blockIdx.x - t.first) * GSR_OPT_CHUNK + wave * (GSR_OPT_CHUNK / 4);
    if (start < t.n) {
        switch (start + GSR_OPT_CHUNK / 4 <= t.n ? t.types : 0) {
#define GSR_OPT_CASE(P, G) case P | G << 4 | GSR_T_ALIGNED: adamw8_blocks<P, G, true, STREAM, 4>(a, t, coef, start); break;
        GSR_OPT_CASE(0, 0) GSR_OPT_CASE(0, 1) GSR_OPT_CASE(0, 2) GSR_OPT_CASE(1, 0) GSR_OPT_CASE(1, 1) GSR_OPT_CASE(1, 2) GSR_OPT_CASE(2, 0) GSR_OPT_CASE(2, 1) GSR_OPT_CASE(2, 2)
#undef GSR_OPT_CASE
        default:
#pragma unroll 1
            for (int b = 0; b < 4; b++)
                if (start + b * GSR_OPT_WINDOW < t.n) adamw8_blocks<0, 0, false, false, 1>(a, t, coef, start + b * GSR_OPT_WINDOW);
        }
    }
    opt_end(a);
}

struct MomentTensor { const uint8_t* rms; const int8_t* ratio; const uint8_t* window; void* exp_avg; void* root; long long n; uint32_t first; int aligned; };
struct MomentArgs { int count; float unit; int type; MomentTensor t[GSR_OPT_MAX]; };

template <int TYPE>
__device__ __forceinline__ void moments_chunk(const MomentArgs& a, const MomentTensor& t, long long base)
{
    if (t.aligned) {
        uint32_t cu[4], cr[4], w[4];
#pragma unroll
        for (int v = 0; v < 4; v++) {
            const long long i = base + 4 * (v * GSR_OPT_THREADS + (int)threadIdx.x);
            cu[v] = cr[v] = w[v] = 0u;
            if (i < t.n) w[v] = t.window[i / GSR_OPT_WINDOW];
            if (i + 4 <= t.n) { cu[v] = *reinterpret_cast<const uint32_t*>(t.rms + i); cr[v] = *reinterpret_cast<const uint32_t*>(t.ratio + i); }
            else for (int k = 0; i + k < t.n; k++) { cu[v] |= (uint32_t)t.rms[i + k] << (8 * k); cr[v] |= (uint32_t)(uint8_t)t.ratio[i + k] << (8 * k); }
        }
#pragma unroll
        for (int v = 0; v < 4; v++) {
            const long long i = base + 4 * (v * GSR_OPT_THREADS + (int)threadIdx.x);
            opt_f4 m, u;
#pragma unroll
            for (int k = 0; k < 4; k++) {
                u[k] = opt_decode((cu[v] >> (8 * k)) & 255u, 16u * w[v] + 1u);
                m[k] = ((float)(int8_t)(cr[v] >> (8 * k)) * a.unit) * u[k];
            }
            if (i + 4 <= t.n) { opt_store4<TYPE, false>(t.exp_avg, i, m); opt_store4<TYPE, false>(t.root, i, u); }
            else
#pragma unroll
                for (int k = 0; k < 4; k++) if (i + k < t.n) { opt_store(t.exp_avg, i + k, TYPE, m[k]); opt_store(t.root, i + k, TYPE, u[k]); }
        }
    } else {
        for (int k = threadIdx.x; k < GSR_OPT_CHUNK && base + k < t.n; k += GSR_OPT_THREADS) {
            const long long i = base + k;
            const float u = opt_decode(t.rms[i], 16u * t.window[i / GSR_OPT_WINDOW] + 1u);
            opt_store(t.exp_avg, i, TYPE, ((float)t.ratio[i] * a.unit) * u);
            opt_store(t.root, i, TYPE, u);
        }
    }
}

__global__ void __launch_bounds__(GSR_OPT_THREADS) k_moments8(MomentArgs a)
{
    const MomentTensor& t = a.t[opt_find(a.t, a.count, blockIdx.x)];
    const long long base = (long long)(blockIdx.x - t.first) * GSR_OPT_CHUNK;
    if (a.type == GSR_T_F32) moments_chunk<GSR_T_F32>(a, t, base);
    else if (a.type == GSR_T_BF16) moments_chunk<GSR_T_BF16>(a, t, base);
    else moments_chunk<GSR_T_F16>(a, t, base);
}

// ---- eviction by accumulated compositing weight ----------------------------------------------------------------------------------
//
// A pixel reads the map as a query reads a cache: splat i with the weight alpha_i T_i.  The rows that stay are the `recent` newest (no
// view has weighed them yet) and, of the others, the k with the largest accumulated weight; ties go to the lowest index, NaN counts as -inf.
// The k-th largest is found exactly by a radix select on order-preserving bit patterns (11 + 11 + 10 bits, one histogram launch each),
// the rows' places by counting per tile of rows; every tensor of the map and of its optimiser is then compacted in one launch.  No
// workgroup ever waits for another: a launch's end is the only barrier between them.

#define GSR_EV_UNITS 16         // units of a lane whose loads are in flight together (4: 178 us for 1.35 M rows of 281 bytes, 8: 173, 16: 159; 32 of twice as large a chunk: 171)
#define GSR_EV_BLOCKS 4         // blocks of codes likewise
#define GSR_EV_CHUNK 8192       // units of one byte that a workgroup copies (of others GSR_OPT_CHUNK)
#define GSR_EV_BINS 2048
#define GSR_EV_COPIES 8         // of the first histogram in LDS: its bins are exponents, a wave's lanes meet in few of them
#define GSR_EV_TILE 1024        // rows of a tile, or a multiple of it
#define GSR_EV_TILES 2048       // tiles at most: every workgroup adds up its predecessors' counts by itself
#define GSR_EV_SMALL 8192       // rows up to which one workgroup does it all (a call at 8192 rows: 21 us for the six launches' 29; with 16 views 27 for 29)

struct EvictArgs {
    int P, views, old, k;       // old = P - recent: the rows that compete; k of them stay
    double decay;
    const float* scores; const float* weights;
    float* total;               // [P] accumulated weights
    uint32_t* hist;             // [3][GSR_EV_BINS]
    uint32_t* found;            // [3][2]: leading bits of the k-th largest key and its rank among those that share them, by level
    uint2* counts;              // [tiles] (above, equal)
    int tile_rows;
    long long* kept; float* scores_out;
};

// The accumulated weights of U rows, summed in the views' order.  No load waits for another: rows behind the end load the last row again,
// views behind the last the last view (a load under a condition is waited for where it stands: k_evict_scores 22 us at 1.5 M rows and 4
// views, 15 so).
template <int U>
__device__ __forceinline__ void evict_scores(const EvictArgs& a, const long long (&i)[U], float (&s)[U])
{
    long long j[U];
    float x[U];
    double w[U];
#pragma unroll
    for (int u = 0; u < U; u++) { j[u] = i[u] < a.P ? i[u] : a.P - 1; x[u] = a.scores[j[u]]; w[u] = 0.0; }
    for (int v = 0; v < a.views; v += 4) {
        float y[4][U];
#pragma unroll
        for (int k = 0; k < 4; k++)
#pragma unroll
            for (int u = 0; u < U; u++) y[k][u] = a.weights[(long long)(v + k < a.views ? v + k : a.views - 1) * a.P + j[u]];
#pragma unroll
        for (int k = 0; k < 4; k++)
            if (v + k < a.views) {
#pragma unroll
                for (int u = 0; u < U; u++) w[u] += (double)y[k][u];
            }
    }
#pragma unroll
    for (int u = 0; u < U; u++) s[u] = (float)((double)x[u] * a.decay + w[u]);
}
__device__ __forceinline__ uint32_t evict_key(float x)          // larger score <=> larger key; NaN as -inf, -0 as +0
{
    if (x != x) x = -__builtin_inff();
    const uint32_t b = __float_as_uint(x + 0.0f);
    return b ^ (b >> 31 ? 0xffffffffu : 0x80000000u);
}
// No key is 0 or 2^32 - 1 (-inf has 0x007fffff, +inf 0xff800000).
#define GSR_EV_NONE 0xffffffffu
#define GSR_EV_ALL 0u

// Which bin, counted from the highest, holds the k-th largest (k >= 1), and its rank among that bin's.  T threads, all of them; NB bins.
template <int T, int NB>
__device__ __forceinline__ void evict_pick(const uint32_t* hist, uint32_t k, uint32_t* s_tmp /*[T / 64 + 2]*/, uint32_t& bin, uint32_t& rank)
{
    constexpr int per = NB / T;
    const int t = threadIdx.x;
    uint32_t c[per], sum = 0;
#pragma unroll
    for (int j = 0; j < per; j++) { c[j] = hist[NB - 1 - (t * per + j)]; sum += c[j]; }
    uint32_t incl = sum;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const uint32_t o = __shfl_up(incl, off, 64);
        if ((t & 63) >= off) incl += o;
    }
    __syncthreads();          // (s_tmp may still be read from a previous pick)
    if ((t & 63) == 63) s_tmp[t >> 6] = incl;
    __syncthreads();
    for (int w = 0; w < (t >> 6); w++) incl += s_tmp[w];
    uint32_t before = incl - sum;
    if (k > before && k <= incl) {
#pragma unroll
        for (int j = 0; j < per; j++) {
            if (k > before && k <= before + c[j]) { s_tmp[T / 64] = (uint32_t)(NB - 1 - (t * per + j)); s_tmp[T / 64 + 1] = k - before; }
            before += c[j];
        }
    }
    __syncthreads();
    bin = s_tmp[T / 64];
    rank = s_tmp[T / 64 + 1];
}

__device__ __forceinline__ uint32_t wave_sum_u32(uint32_t v)          // over 64 lanes, in every lane (DPP)
{
#define GSR_DPP_SUM(ctrl, rm) v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, ctrl, rm, 0xf, true);
    GSR_DPP_SUM(0x111, 0xf) GSR_DPP_SUM(0x112, 0xf) GSR_DPP_SUM(0x114, 0xf) GSR_DPP_SUM(0x118, 0xf) GSR_DPP_SUM(0x142, 0xa) GSR_DPP_SUM(0x143, 0xc)
#undef GSR_DPP_SUM
    return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}

// Launch 1: the accumulated weights and the histogram of their keys' upper 11 bits.
__global__ void __launch_bounds__(512) k_evict_scores(EvictArgs a)
{
    __shared__ uint32_t s_hist[GSR_EV_COPIES * (GSR_EV_BINS + 1)];          // (a bin's copies in banks of their own)
    for (int b = threadIdx.x; b < GSR_EV_COPIES * (GSR_EV_BINS + 1); b += 512) s_hist[b] = 0u;
    __syncthreads();
    uint32_t* const own = s_hist + (threadIdx.x & (GSR_EV_COPIES - 1)) * (GSR_EV_BINS + 1);
    const long long step = (long long)gridDim.x * 2048;
    for (long long i0 = (long long)blockIdx.x * 2048 + threadIdx.x; i0 < a.P; i0 += step) {
        const long long i[4] = {i0, i0 + 512, i0 + 1024, i0 + 1536};
        float s[4];
        evict_scores(a, i, s);
#pragma unroll
        for (int u = 0; u < 4; u++) {
            if (i[u] < a.P) a.total[i[u]] = s[u];
            if (i[u] < a.old) atomicAdd(&own[evict_key(s[u]) >> 21], 1u);
        }
    }
    __syncthreads();
    for (int b = threadIdx.x; b < GSR_EV_BINS; b += 512) {
        uint32_t n = 0;
#pragma unroll
        for (int c = 0; c < GSR_EV_COPIES; c++) n += s_hist[c * (GSR_EV_BINS + 1) + b];
        if (n) atomicAdd(&a.hist[b], n);
    }
}

// Launches 2 and 3: the histogram of the next bits among the keys that share the k-th largest's leading ones.  Few, large workgroups:
// each flushes up to 2048 bins with global atomics (1024 workgroups of 256: 18 us at 1.5 M rows).
template <int LEVEL>
__global__ void __launch_bounds__(1024) k_evict_hist(EvictArgs a)
{
    __shared__ uint32_t s_hist[GSR_EV_BINS];
    __shared__ uint32_t s_tmp[1024 / 64 + 2];
    constexpr int NB = LEVEL == 2 ? GSR_EV_BINS : GSR_EV_BINS / 2;
    for (int b = threadIdx.x; b < NB; b += 1024) s_hist[b] = 0u;
    uint32_t prefix, rank;
    if (LEVEL == 2) evict_pick<1024, GSR_EV_BINS>(a.hist, (uint32_t)a.k, s_tmp, prefix, rank);
    else {
        uint32_t bin;
        evict_pick<1024, GSR_EV_BINS>(a.hist + GSR_EV_BINS, a.found[1], s_tmp, bin, rank);
        prefix = (a.found[0] << 11) | bin;
    }
    if (blockIdx.x == 0 && threadIdx.x == 0) { a.found[2 * (LEVEL - 2)] = prefix; a.found[2 * (LEVEL - 2) + 1] = rank; }
    const long long step = (long long)gridDim.x * 8192;
    for (long long i0 = (long long)blockIdx.x * 8192 + threadIdx.x; i0 < a.old; i0 += step) {
        float x[8];
#pragma unroll
        for (int u = 0; u < 8; u++) x[u] = a.total[i0 + 1024 * u < a.old ? i0 + 1024 * u : a.old - 1];
#pragma unroll
        for (int u = 0; u < 8; u++) {
            const uint32_t key = evict_key(x[u]);
            if (i0 + 1024 * u >= a.old) break;
            if (LEVEL == 2) { if ((key >> 21) == prefix) atomicAdd(&s_hist[(key >> 10) & 2047u], 1u); }
            else            { if ((key >> 10) == prefix) atomicAdd(&s_hist[key & 1023u], 1u); }
        }
    }
    __syncthreads();
    for (int b = threadIdx.x; b < NB; b += 1024)
        if (s_hist[b]) atomicAdd(&a.hist[(LEVEL - 1) * GSR_EV_BINS + b], s_hist[b]);
}

// Launch 4: the smallest key that stays and how many rows with exactly that key do; how many of either kind each tile has.
__global__ void __launch_bounds__(256) k_evict_count(EvictArgs a)
{
    __shared__ uint32_t s_tmp[256 / 64 + 2];
    __shared__ uint32_t s_n[2];
    uint32_t key, ties = 0u;
    if (a.k == 0) key = GSR_EV_NONE;
    else if (a.k == a.old) key = GSR_EV_ALL;
    else {
        evict_pick<256, GSR_EV_BINS / 2>(a.hist + 2 * GSR_EV_BINS, a.found[3], s_tmp, key, ties);
        key |= a.found[2] << 10;
    }
    if (blockIdx.x == 0 && threadIdx.x == 0) { a.found[4] = key; a.found[5] = ties; }
    if (threadIdx.x < 2) s_n[threadIdx.x] = 0u;
    __syncthreads();
    uint32_t above = 0, equal = 0;
    const long long lo = (long long)blockIdx.x * a.tile_rows;
    for (int r0 = 0; r0 < a.tile_rows; r0 += 1024) {
        float x[4];
        if (r0 + 1024 <= a.tile_rows && lo + r0 + 1024 <= a.old) {
#pragma unroll
            for (int u = 0; u < 4; u++) x[u] = a.total[lo + r0 + 256 * u + threadIdx.x];
#pragma unroll
            for (int u = 0; u < 4; u++) { above += evict_key(x[u]) > key; equal += evict_key(x[u]) == key; }
        } else {
            for (int r = r0 + (int)threadIdx.x; r < a.tile_rows && lo + r < a.old && r < r0 + 1024; r += 256) { const uint32_t k = evict_key(a.total[lo + r]); above += k > key; equal += k == key; }
        }
    }
    above = wave_sum_u32(above); equal = wave_sum_u32(equal);
    if ((threadIdx.x & 63) == 0) { atomicAdd(&s_n[0], above); atomicAdd(&s_n[1], equal); }
    __syncthreads();
    if (threadIdx.x == 0) a.counts[blockIdx.x] = make_uint2(s_n[0], s_n[1]);
}

// The rows of one pass that stay, written in order: thread t has rows lo + T u + t, u < U; `above`, `equal`: how many were counted before `lo`,
// advanced.  Two barriers; s_n [U * T / 64].
template <int T, int U>
__device__ __forceinline__ void evict_emit_pass(const EvictArgs& a, long long lo, const float (&s)[U], int rows, uint32_t key, uint32_t ties,
                                                uint2* s_n, uint32_t& above, uint32_t& equal)
{
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    unsigned long long ma[U], me[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
        const int r = T * u + t;
        const bool in = r < rows && lo + r < a.old;
        const uint32_t x = evict_key(s[u]);
        ma[u] = __ballot(in && x > key); me[u] = __ballot(in && x == key);
        if (lane == 0) s_n[u * (T / 64) + wave] = make_uint2((uint32_t)__popcll(ma[u]), (uint32_t)__popcll(me[u]));
    }
    __syncthreads();
    const unsigned long long below = (1ull << lane) - 1ull;
    uint32_t na = above, ne = equal;
#pragma unroll
    for (int u = 0; u < U; u++) {
#pragma unroll
        for (int w = 0; w < T / 64; w++) {
            if (w == wave) {
                const int r = T * u + t;
                const long long i = lo + r;
                const uint32_t ia = na + (uint32_t)__popcll(ma[u] & below), ie = ne + (uint32_t)__popcll(me[u] & below);
                long long at = -1;
                if (r < rows && i >= a.old) at = (long long)a.k + (i - a.old);
                else if ((ma[u] >> lane) & 1ull || ((me[u] >> lane) & 1ull && ie < ties)) at = (long long)ia + (ie < ties ? ie : ties);
                if (at >= 0) { a.kept[at] = i; a.scores_out[at] = s[u]; }
            }
            const uint2 n = s_n[u * (T / 64) + w];
            na += n.x; ne += n.y;
        }
    }
    above = na; equal = ne;
    __syncthreads();
}

// Launch 5: the rows that stay, in their order.
__global__ void __launch_bounds__(256) k_evict_emit(EvictArgs a)
{
    __shared__ uint2 s_n[16];
    __shared__ uint32_t s_base[2];
    const int t = threadIdx.x;
    const long long lo = (long long)blockIdx.x * a.tile_rows;
    const int rows = (int)(a.P - lo < a.tile_rows ? a.P - lo : a.tile_rows);
    float s[4];
    const auto read = [&](int r0) {
#pragma unroll
        for (int u = 0; u < 4; u++) s[u] = a.total[lo + (r0 + 256 * u + t < rows ? r0 + 256 * u + t : 0)];
    };
    read(0);
    if (t < 2) s_base[t] = 0u;
    __syncthreads();
    uint32_t above = 0, equal = 0;          // of the tiles in front
    {
        uint2 n[GSR_EV_TILES / 256];
#pragma unroll
        for (int j = 0; j < GSR_EV_TILES / 256; j++) n[j] = a.counts[256 * j + t < (int)blockIdx.x ? 256 * j + t : 0];
#pragma unroll
        for (int j = 0; j < GSR_EV_TILES / 256; j++) if (256 * j + t < (int)blockIdx.x) { above += n[j].x; equal += n[j].y; }
    }
    above = wave_sum_u32(above); equal = wave_sum_u32(equal);
    if ((t & 63) == 0) { atomicAdd(&s_base[0], above); atomicAdd(&s_base[1], equal); }
    const uint32_t key = a.found[4], ties = a.found[5];
    __syncthreads();
    above = s_base[0]; equal = s_base[1];
    for (int r0 = 0; r0 < rows; r0 += GSR_EV_TILE) {
        if (r0) read(r0);
        evict_emit_pass<256, 4>(a, lo + r0, s, rows - r0, key, ties, s_n, above, equal);
    }
}

// All of it for a small map: scores in registers, histograms in LDS.
__global__ void __launch_bounds__(1024) k_evict_small(EvictArgs a)
{
    constexpr int U = GSR_EV_SMALL / 1024;
    __shared__ uint32_t s_hist[GSR_EV_BINS];
    __shared__ uint32_t s_tmp[1024 / 64 + 2];
    __shared__ uint2 s_n[16 * U];
    const int t = threadIdx.x;
    long long i[U];
    float s[U];
#pragma unroll
    for (int u = 0; u < U; u++) i[u] = 1024 * u + t;
    evict_scores(a, i, s);
    uint32_t key = GSR_EV_NONE, ties = 0u;
    if (a.k > 0 && a.k == a.old) key = GSR_EV_ALL;
    else if (a.k > 0) {
        uint32_t prefix = 0u, rank = (uint32_t)a.k, bin;
#pragma unroll 1
        for (int level = 0; level < 3; level++) {          // 11, 11 and 10 bits (the last histogram's upper half stays empty)
            const int shift = level == 0 ? 21 : level == 1 ? 10 : 0, known = level == 0 ? 0 : level == 1 ? 21 : 10;
            __syncthreads();
            s_hist[t] = 0u; s_hist[1024 + t] = 0u;
            __syncthreads();
#pragma unroll
            for (int u = 0; u < U; u++) {
                const uint32_t x = evict_key(s[u]);
                if (1024 * u + t < a.old && (level == 0 || (x >> known) == prefix)) atomicAdd(&s_hist[(x >> shift) & (level == 2 ? 1023u : 2047u)], 1u);
            }
            __syncthreads();
            evict_pick<1024, GSR_EV_BINS>(s_hist, rank, s_tmp, bin, rank);
            prefix = level == 2 ? (prefix << 10) | bin : (prefix << 11) | bin;
        }
        key = prefix; ties = rank;
    }
    uint32_t above = 0, equal = 0;
    evict_emit_pass<1024, U>(a, 0, s, a.P, key, ties, s_n, above, equal);
}

struct RowTensor {
    const void* src; void* dst;
    const uint8_t* src_window; uint8_t* dst_window;          // codes of the 8-bit root: their windows (then a row's unit is one code)
    long long row;              // units of a row
    uint32_t first;             // its first workgroup
    uint32_t magic;             // floor(x / row) = x magic / 2^32 for x < row + GSR_EV_CHUNK; 0: a row of one, or too long for that
    int unit;                   // bytes of a unit: 1, 2, 4, 8 or 16
    int large;                  // the source has 4 GB or more
};
struct RowArgs { int count; long long keep; const long long* kept; RowTensor t[GSR_OPT_MAX]; };

// Where the units of a chunk come from: its first unit's row and column by one division, the others' by a multiplication.  OFF: the type of
// the sources' byte offsets.
template <class OFF>
struct RowWalk {
    const char* kept; OFF row_bytes; uint32_t row, col0, magic, last;          // kept: of the chunk's first row on; last: the chunk's last unit
    __device__ __forceinline__ RowWalk(const RowArgs& a, const RowTensor& t, long long base, uint32_t chunk)
    {
        const long long left = a.keep * t.row - base, row0 = base / t.row;
        kept = reinterpret_cast<const char*>(a.kept + row0); row = (uint32_t)t.row; magic = t.magic;
        row_bytes = (OFF)t.row * (OFF)t.unit;
        col0 = (uint32_t)(base - row0 * t.row);
        last = left < chunk ? (uint32_t)left - 1u : chunk - 1u;
    }
    __device__ __forceinline__ uint32_t place(uint32_t x, uint32_t& col) const          // which row of the chunk's, and which unit in it
    {
        const uint32_t y = col0 + (x < last ? x : last);          // (behind the end: the last one again, not stored)
        const uint32_t q = magic ? __umulhi(y, magic) : row == 1 ? y : y / row;
        col = y - q * row;
        return q;
    }
    __device__ __forceinline__ OFF number(uint32_t q) const          // of the chunk's q-th row (int64 in memory, of a chunk under 2^32 bytes)
    {
        return (OFF)*reinterpret_cast<const OFF*>(kept + (uint32_t)(8u * q));
    }
    // The sources of U units: all their rows' numbers are loaded before the first is used.
    template <int UNIT, int U>
    __device__ __forceinline__ void from(const uint32_t (&x)[U], OFF (&e)[U]) const
    {
        uint32_t col[U];
#pragma unroll
        for (int u = 0; u < U; u++) e[u] = number(place(x[u], col[u]));
#pragma unroll
        for (int u = 0; u < U; u++) e[u] = e[u] * row_bytes + (OFF)(col[u] * UNIT);
    }
    // The same for groups of four consecutive bytes of rows of three or more, which lie in two rows at most: one division, two loads and two
    // products a group.  wrap: this unit is in the second row.
    template <int U>
    __device__ __forceinline__ void fours(const uint32_t (&x)[U], OFF (&e)[U], bool (&wrap)[U]) const
    {
        uint32_t q[U / 4], col[U / 4];
        OFF first[U / 4], second[U / 4];
#pragma unroll
        for (int j = 0; j < U / 4; j++) q[j] = place(x[4 * j], col[j]);
#pragma unroll
        for (int j = 0; j < U / 4; j++) { first[j] = number(q[j]); second[j] = number(q[j] + (col[j] + 3 >= row ? 1 : 0)); }
#pragma unroll
        for (int j = 0; j < U / 4; j++) { first[j] = first[j] * row_bytes + col[j]; second[j] = second[j] * row_bytes + (OFF)col[j] - (OFF)row; }
#pragma unroll
        for (int u = 0; u < U; u++) { wrap[u] = col[u / 4] + (u & 3) >= row; e[u] = (wrap[u] ? second[u / 4] : first[u / 4]) + (OFF)(u & 3); }
    }
};

// Consecutive lanes, consecutive units, GSR_EV_UNITS of a lane in flight; nothing is loaded under a condition, which would have each load
// waited for where it stands (250 us for 1.35 M rows of 281 bytes, 159 so: 776 MB at 4.9 TB/s).  Staging the source's span in LDS, evicted
// rows with it, was slower (280), a workgroup per 256 rows of all tensors as well (166).
template <class T>
__device__ __forceinline__ void evict_chunk(const RowArgs& a, const RowTensor& t, long long base, uint32_t chunk)
{
    constexpr int U = sizeof(T) <= 4 ? GSR_EV_UNITS : GSR_EV_UNITS * 4 / (int)sizeof(T);          // the same bytes, and registers, for every unit
    typedef unsigned long long OFF;          // (no register is scarce here: 32 bits gain nothing)
    const RowWalk<OFF> w(a, t, base, chunk);
    const char* src = static_cast<const char*>(t.src);
    T* dst = static_cast<T*>(t.dst) + base;
#pragma unroll 1
    for (int h = 0; h < GSR_OPT_CHUNK / GSR_OPT_THREADS; h += U) {
        uint32_t x[U];
        OFF e[U];
        T v[U];
#pragma unroll
        for (int u = 0; u < U; u++) x[u] = (h + u) * GSR_OPT_THREADS + threadIdx.x;
        w.template from<(int)sizeof(T)>(x, e);
#pragma unroll
        for (int u = 0; u < U; u++) v[u] = *reinterpret_cast<const T*>(src + e[u]);
#pragma unroll
        for (int u = 0; u < U; u++) if (x[u] <= w.last) dst[x[u]] = v[u];
    }
}

// Units of one byte: four consecutive ones per lane, a wave per 256, GSR_EV_BLOCKS of those in flight; offsets of 32 bits where the source
// has less than 4 GB (1.35 M rows of 180 bytes: 205 us, 240 with 64; as codes 240, 294).
//
// Codes of the 8-bit root change their block with their row: the float's upper bits move into the new block's window, exactly, but for
// what lies under that window (raised to its lowest value).  The ratios are tensors of their own and copied as they are, so a raised
// row's next update is what it would have been (m / sqrt(v) is the ratio either way), and the momentum that its bytes stand for grows with the root.
template <bool CODES, class OFF>
__device__ __forceinline__ void evict_bytes(const RowArgs& a, const RowTensor& t, long long base, uint32_t chunk)
{
    const RowWalk<OFF> w(a, t, base, chunk);
    const int lane = threadIdx.x & 63;
    const uint8_t* src = static_cast<const uint8_t*>(t.src);
    uint8_t* dst = static_cast<uint8_t*>(t.dst) + base;
#pragma unroll 1
    for (uint32_t b = threadIdx.x >> 6; b * GSR_OPT_WINDOW <= w.last; b += 4 * GSR_EV_BLOCKS) {
        constexpr int U = 4 * GSR_EV_BLOCKS;
        uint32_t x[U], v[U], window[U];
        OFF e[U];
#pragma unroll
        for (int k = 0; k < U; k++) x[k] = (b + 4 * (k >> 2)) * GSR_OPT_WINDOW + 4 * lane + (k & 3);
        if (w.row >= 3 && (b + U) * GSR_OPT_WINDOW <= w.last + 1u) {
            // Rows ascend, so four units' sources do: the four bytes from the first and the four up to the last lie inside the tensor and hold them all.
            uint32_t lo[GSR_EV_BLOCKS], hi[GSR_EV_BLOCKS];
            bool wrap[U];
            w.fours(x, e, wrap);
#pragma unroll
            for (int j = 0; j < GSR_EV_BLOCKS; j++) { __builtin_memcpy(&lo[j], src + e[4 * j], 4); __builtin_memcpy(&hi[j], src + (e[4 * j + 3] - 3), 4); }
#pragma unroll
            for (int k = 0; k < U; k++) v[k] = ((wrap[k] ? hi[k / 4] : lo[k / 4]) >> (8 * (k & 3))) & 255u;
        } else {
            w.template from<1>(x, e);
#pragma unroll
            for (int k = 0; k < U; k++) v[k] = src[e[k]];
        }
#pragma unroll
        for (int k = 0; k < U; k++) window[k] = CODES ? t.src_window[e[k] / GSR_OPT_WINDOW] : 0u;
#pragma unroll
        for (int j = 0; j < GSR_EV_BLOCKS; j++) {
            const uint32_t at = x[4 * j];
            uint32_t bytes = 0;
            if (CODES) {
                uint32_t top[4], most = 0;
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    top[k] = v[4 * j + k] && x[4 * j + k] <= w.last ? v[4 * j + k] + 16u * window[4 * j + k] + 1u : 0u;
                    most = top[k] > most ? top[k] : most;
                }
                const uint32_t nw = opt_window(wave_max_u32(most) << 19), now = 16u * nw + 1u;
#pragma unroll
                for (int k = 0; k < 4; k++) bytes |= (top[k] == 0u ? 0u : top[k] > now + 1u ? top[k] - now : 1u) << (8 * k);
                if (lane == 0 && at <= w.last) t.dst_window[(base + at) / GSR_OPT_WINDOW] = (uint8_t)nw;
            } else {
#pragma unroll
                for (int k = 0; k < 4; k++) bytes |= v[4 * j + k] << (8 * k);
            }
            if (at + 3 <= w.last && opt_aligned4(dst)) *reinterpret_cast<uint32_t*>(dst + at) = bytes;
            else for (int k = 0; k < 4; k++) if (at + k <= w.last) dst[at + k] = (uint8_t)(bytes >> (8 * k));
        }
    }
}

__global__ void __launch_bounds__(GSR_OPT_THREADS) k_evict_rows(RowArgs a)
{
    const RowTensor& t = a.t[opt_find(a.t, a.count, blockIdx.x)];
    const uint32_t chunk = t.unit == 1 ? GSR_EV_CHUNK : GSR_OPT_CHUNK;
    const long long base = (long long)(blockIdx.x - t.first) * chunk;
    if (t.src_window) { if (t.large) evict_bytes<true, unsigned long long>(a, t, base, chunk); else evict_bytes<true, uint32_t>(a, t, base, chunk); }
    else if (t.unit == 16) evict_chunk<opt_f4>(a, t, base, chunk);
    else if (t.unit == 8) evict_chunk<opt_u2>(a, t, base, chunk);
    else if (t.unit == 4) evict_chunk<uint32_t>(a, t, base, chunk);
    else if (t.unit == 2) evict_chunk<uint16_t>(a, t, base, chunk);
    else if (t.large) evict_bytes<false, unsigned long long>(a, t, base, chunk);
    else evict_bytes<false, uint32_t>(a, t, base, chunk);
}

}  // namespace gsr
