// gsr_mapopt.h -- the optimiser step of a Gaussian map and the pruning that goes with it: what gaussian_splatting/train.py:149-157 leaves
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

enum { GSR_T_F32 = 0, GSR_T_BF16 = 1, GSR_T_F16 = 2 };

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

// ---- the norm of the gradients --------------------------------------------------------------------------------------------------

struct NormTensor { const void* g; long long n; uint32_t first; int type; };          // first: its first chunk in the launch
struct NormArgs {
    int count;
    uint32_t chunks;
    double* partial;            // one sum per workgroup
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

__global__ void __launch_bounds__(GSR_OPT_THREADS) k_grad_norm(NormArgs a)
{
    __shared__ double s[4];
    double sum = 0.0;          // a product of two floats is exact in a double: one rounding per element, 2^-53 of the running sum
    for (uint32_t c = blockIdx.x; c < a.chunks; c += gridDim.x) {
        const NormTensor& t = a.t[opt_find(a.t, a.count, c)];
        const long long base = (long long)(c - t.first) * GSR_OPT_CHUNK;
        for (int k = threadIdx.x; k < GSR_OPT_CHUNK; k += GSR_OPT_THREADS)
            if (base + k < t.n) { const double x = opt_load(t.g, base + k, t.type); sum = __builtin_fma(x, x, sum); }
    }
    sum = opt_block_sum(sum, s);
    if (threadIdx.x == 0) a.partial[blockIdx.x] = sum;
}

// The partial sums in a fixed order (the result does not depend on which workgroup ran when), then torch.nn.utils.clip_grad_norm_'s
// coefficient: min(1, max_norm / (norm + 1e-6)), a NaN norm stays one.
__global__ void __launch_bounds__(GSR_OPT_THREADS) k_grad_norm_finish(const double* __restrict__ partial, int n, float max_norm, float* __restrict__ out)
{
    __shared__ double s[4];
    double sum = 0.0;
    for (int i = threadIdx.x; i < n; i += GSR_OPT_THREADS) sum += partial[i];
    sum = opt_block_sum(sum, s);
    if (threadIdx.x == 0) {
        const float norm = (float)sqrt(sum);
        const float c = max_norm / (norm + 1e-6f);
        out[0] = norm;
        out[1] = c > 1.0f ? 1.0f : c;
    }
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
    uint32_t first;             // first chunk in the launch
    uint32_t key;               // 8 bits: seed and place in the list
    int types;                  // parameter | gradient << 4
};
struct OptArgs {
    int count;
    uint32_t chunks;
    double beta1, beta2;
    float b1, b2, c1, c2, eps;  // (c = 1 - beta)
    float unit, per_unit;       // 8 bits: the ratio's step, and steps per one
    const float* clip;          // nullable: (norm, coefficient)
    OptTensor t[GSR_OPT_MAX];
};

struct OptRates { float shrink, rate, unbias; uint32_t step; };
__device__ __forceinline__ OptRates opt_rates(const OptArgs& a, const OptTensor& t)
{
    const double lr = t.lr_device ? *t.lr_device : t.lr;
    const double b1t = t.clock[0] * a.beta1, b2t = t.clock[1] * a.beta2;
    OptRates r;
    r.shrink = (float)(1.0 - lr * t.decay);
    r.rate = (float)((1.0 / (1.0 - b1t)) * lr);
    r.unbias = (float)(1.0 / sqrt(1.0 - b2t));
    r.step = (uint32_t)(t.clock[2] + 1.0);
    return r;
}

// Every workgroup has read the clocks before it draws a ticket, so the one that draws the last may advance them: the step counts live
// on the device (a captured graph goes on counting) without a launch of their own.  The ticket is the fourth word of the launch's first
// clock and is zero between launches.
__device__ __forceinline__ void opt_advance(const OptArgs& a)
{
    __shared__ int s_last;
    __syncthreads();
    if (threadIdx.x == 0) {
        __threadfence();
        s_last = atomicAdd(reinterpret_cast<unsigned*>(a.t[0].clock + 3), 1u) == gridDim.x - 1u;
    }
    __syncthreads();
    if (!s_last) return;
    for (int i = threadIdx.x; i < a.count; i += GSR_OPT_THREADS) {
        double* c = a.t[i].clock;
        c[0] *= a.beta1; c[1] *= a.beta2; c[2] += 1.0;
        if (i == 0) c[3] = 0.0;
    }
}

__global__ void __launch_bounds__(GSR_OPT_THREADS) k_adamw(OptArgs a)
{
    const float coef = a.clip ? a.clip[1] : 1.0f;
    for (uint32_t c = blockIdx.x; c < a.chunks; c += gridDim.x) {
        const OptTensor& t = a.t[opt_find(a.t, a.count, c)];
        const OptRates r = opt_rates(a, t);
        const long long base = (long long)(c - t.first) * GSR_OPT_CHUNK;
        float* m = static_cast<float*>(t.s0);
        float* v = static_cast<float*>(t.s1);
        for (int k = threadIdx.x; k < GSR_OPT_CHUNK && base + k < t.n; k += GSR_OPT_THREADS) {
            const long long i = base + k;
            const float g = opt_load(t.g, i, t.types >> 4) * coef;
            const float m1 = m[i] * a.b1 + g * a.c1;
            const float v1 = v[i] * a.b2 + (g * g) * a.c2;
            const float p = opt_load(t.p, i, t.types & 15) * r.shrink - (m1 / (sqrtf(v1) * r.unbias + a.eps)) * r.rate;
            m[i] = m1; v[i] = v1;
            opt_store(t.p, i, t.types & 15, p);
        }
    }
    opt_advance(a);
}

// ---- AdamW with a byte for each moment -------------------------------------------------------------------------------------------
//
// Stored are u = sqrt(v) and r = m / u.
//   u   the upper 13 bits of the float (sign, exponent, four bits of mantissa), minus 16 w + 1, in a byte; w, one byte per 256 elements,
//       places the window: sixteen binades under the block's largest root.  0 stands for 0; what is positive but lies under the window is
//       raised to code 1 (a smaller update, never a larger one).  Rounding is stochastic (19 random bits added under the kept ones: exactly
//       unbiased inside a binade): with beta2 = 0.999 the moment moves by 0.1 % per step, and rounded to the nearest sixteenth it
//       would stand still wherever it once was.
//   r   |m| <= B sqrt(v) whatever the gradients were, B = (1 - b1) / sqrt((1 - b2)(1 - b1^2 / b2)) (Cauchy-Schwarz over the two
//       exponential sums; 7.27 for 0.9 / 0.999): 127 steps of B / 127 to either side, stochastic (13 bits).  A momentum quantised for
//       itself could meet a root that its own block has rounded to almost nothing, and with train.py's eps = 1e-15 the quotient would
//       throw the splat across the scene; the ratio is the update, and cannot.
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
__device__ __forceinline__ uint32_t wave_max_u32(uint32_t v)
{
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) { const uint32_t o = (uint32_t)__shfl_xor((int)v, off, 64); v = o > v ? o : v; }
    return v;
}
__device__ __forceinline__ uint32_t opt_window(uint32_t largest)          // of the block's largest finite root, by its bits
{
    const int w = (int)(largest >> 23) - 15;          // its binade is the last but one: rounding up may need the next one's first value
    return w > 0 ? (uint32_t)w : 0u;
}

__global__ void __launch_bounds__(GSR_OPT_THREADS) k_adamw8(OptArgs a)
{
    const float coef = a.clip ? a.clip[1] : 1.0f;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (uint32_t c = blockIdx.x; c < a.chunks; c += gridDim.x) {
        const OptTensor& t = a.t[opt_find(a.t, a.count, c)];
        const OptRates r = opt_rates(a, t);
        const uint32_t key = opt_mix(t.key + r.step);
        uint8_t* rms = static_cast<uint8_t*>(t.s0);
        int8_t* ratio = static_cast<int8_t*>(t.s1);
        for (int b = wave; b < GSR_OPT_CHUNK / GSR_OPT_WINDOW; b += 4) {
            const long long start = (long long)(c - t.first) * GSR_OPT_CHUNK + b * GSR_OPT_WINDOW;
            if (start >= t.n) break;          // (the whole wave)
            const long long i0 = start + 4 * lane;
            const uint32_t old = 16u * t.window[start / GSR_OPT_WINDOW] + 1u;
            float m1[4], u1[4];
            uint32_t top = 0;
#pragma unroll
            for (int k = 0; k < 4; k++) {
                m1[k] = u1[k] = 0.0f;
                if (i0 + k < t.n) {
                    const float u = opt_decode(rms[i0 + k], old);
                    const float g = opt_load(t.g, i0 + k, t.types >> 4) * coef;
                    m1[k] = (((float)ratio[i0 + k] * a.unit) * u) * a.b1 + g * a.c1;
                    u1[k] = sqrtf((u * u) * a.b2 + (g * g) * a.c2);
                    const float p = opt_load(t.p, i0 + k, t.types & 15) * r.shrink - (m1[k] / (u1[k] * r.unbias + a.eps)) * r.rate;
                    opt_store(t.p, i0 + k, t.types & 15, p);
                    const uint32_t bits = __float_as_uint(u1[k]) & 0x7fffffffu;
                    if (bits < 0x7f800000u && bits > top) top = bits;          // (an infinite root or a NaN leaves its neighbours' window alone)
                }
            }
            const uint32_t w = opt_window(wave_max_u32(top)), now = 16u * w + 1u;
            const uint32_t j = (uint32_t)(i0 >> 2), jh = (uint32_t)(i0 >> 34);
            const uint32_t h = opt_mix(((j * 0x9E3779B1u) ^ key) + jh * 0x85EBCA77u);
#pragma unroll
            for (int k = 0; k < 4; k++) {
                if (i0 + k >= t.n) break;
                const uint32_t d = opt_dither(h, k);
                const uint32_t bits = __float_as_uint(u1[k]) & 0x7fffffffu;
                int code = (int)((bits + (d >> 13)) >> 19) - (int)now;
                code = code < 1 ? 1 : (code > 255 ? 255 : code);
                if (bits >= 0x7f800000u) code = 255;
                if (bits == 0u) code = 0;
                const float u = opt_decode((uint32_t)code, now);
                float q = floorf((m1[k] / u) * a.per_unit + (float)(d & 8191u) * (1.0f / 8192.0f));
                q = q < -127.0f ? -127.0f : (q > 127.0f ? 127.0f : q);
                if (!(u > 0.0f) || q != q) q = 0.0f;
                rms[i0 + k] = (uint8_t)code;
                ratio[i0 + k] = (int8_t)q;
            }
            if (lane == 0) t.window[start / GSR_OPT_WINDOW] = (uint8_t)w;
        }
    }
    opt_advance(a);
}

struct MomentTensor { const uint8_t* rms; const int8_t* ratio; const uint8_t* window; void* exp_avg; void* root; long long n; uint32_t first; };
struct MomentArgs { int count; uint32_t chunks; float unit; int type; MomentTensor t[GSR_OPT_MAX]; };

__global__ void __launch_bounds__(GSR_OPT_THREADS) k_moments8(MomentArgs a)
{
    for (uint32_t c = blockIdx.x; c < a.chunks; c += gridDim.x) {
        const MomentTensor& t = a.t[opt_find(a.t, a.count, c)];
        const long long base = (long long)(c - t.first) * GSR_OPT_CHUNK;
        for (int k = threadIdx.x; k < GSR_OPT_CHUNK && base + k < t.n; k += GSR_OPT_THREADS) {
            const long long i = base + k;
            const float u = opt_decode(t.rms[i], 16u * t.window[i / GSR_OPT_WINDOW] + 1u);
            opt_store(t.exp_avg, i, a.type, ((float)t.ratio[i] * a.unit) * u);
            opt_store(t.root, i, a.type, u);
        }
    }
}

// ---- eviction by accumulated compositing weight ----------------------------------------------------------------------------------
//
// A pixel reads the map as a query reads a cache: splat i with the weight alpha_i T_i.  The rows that stay are the `recent` newest (no
// view has weighed them yet) and, of the others, the k with the largest accumulated weight; ties go to the lowest index, NaN counts as -inf.
// The k-th largest is found exactly by a radix select on order-preserving bit patterns (11 + 11 + 10 bits, one histogram launch each),
// the rows' places by counting per tile of rows; every tensor of the map and of its optimiser is then compacted in one launch.

#define GSR_EV_BINS 2048
#define GSR_EV_TILES 1024       // tiles of rows: few enough for every workgroup to add up its predecessors' counts by itself

struct EvictArgs {
    int P, views, old, k;       // old = P - recent: the rows that compete; k of them stay
    double decay;
    const float* scores; const float* weights;
    float* total;               // [P] accumulated weights
    uint32_t* hist;             // [3][GSR_EV_BINS]
    uint2* counts;              // [tiles] (above, equal)
    int tiles, tile_rows;
    long long* kept; float* scores_out;
};

__device__ __forceinline__ uint32_t evict_key(float x)          // larger score <=> larger key; NaN as -inf, -0 as +0
{
    if (x != x) x = -__builtin_inff();
    const uint32_t b = __float_as_uint(x + 0.0f);
    return b ^ (b >> 31 ? 0xffffffffu : 0x80000000u);
}

// Which bin, counted from the highest, holds the k-th largest (k >= 1), and its rank among that bin's.  256 threads, nb = 256 * per.
__device__ __forceinline__ void evict_pick(const uint32_t* __restrict__ hist, int per, uint32_t k, uint32_t* s_tmp /*[8]*/, uint32_t& bin, uint32_t& k_rem)
{
    const int t = threadIdx.x, nb = 256 * per;
    uint32_t c[8], sum = 0;
    for (int j = 0; j < per; j++) { c[j] = hist[nb - 1 - (t * per + j)]; sum += c[j]; }
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
        int j = 0;
        while (j < per - 1 && k > before + c[j]) { before += c[j]; j++; }
        s_tmp[4] = (uint32_t)(nb - 1 - (t * per + j));
        s_tmp[5] = k - before;
    }
    __syncthreads();
    bin = s_tmp[4];
    k_rem = s_tmp[5];
}

__device__ __forceinline__ void evict_flush(const uint32_t* s_hist, uint32_t* __restrict__ hist, int nb)
{
    __syncthreads();
    for (int b = threadIdx.x; b < nb; b += 256)
        if (s_hist[b]) atomicAdd(&hist[b], s_hist[b]);
}

__global__ void __launch_bounds__(256) k_evict_scores(EvictArgs a)
{
    __shared__ uint32_t s_hist[GSR_EV_BINS];
    for (int b = threadIdx.x; b < GSR_EV_BINS; b += 256) s_hist[b] = 0u;
    __syncthreads();
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < a.P; i += (long long)gridDim.x * 256) {
        double x = (double)a.scores[i] * a.decay;
        double w = 0.0;
        for (int v = 0; v < a.views; v++) w += (double)a.weights[(long long)v * a.P + i];
        const float s = (float)(x + w);
        a.total[i] = s;
        if (i < a.old) atomicAdd(&s_hist[evict_key(s) >> 21], 1u);
    }
    evict_flush(s_hist, a.hist, GSR_EV_BINS);
}

template <int LEVEL>
__global__ void __launch_bounds__(256) k_evict_hist(EvictArgs a)
{
    __shared__ uint32_t s_hist[GSR_EV_BINS];
    __shared__ uint32_t s_tmp[8];
    constexpr int NB = LEVEL == 2 ? GSR_EV_BINS : GSR_EV_BINS / 2;
    for (int b = threadIdx.x; b < NB; b += 256) s_hist[b] = 0u;
    uint32_t prefix, k;
    evict_pick(a.hist, GSR_EV_BINS / 256, (uint32_t)a.k, s_tmp, prefix, k);
    if (LEVEL == 3) {
        uint32_t bin;
        evict_pick(a.hist + GSR_EV_BINS, GSR_EV_BINS / 256, k, s_tmp, bin, k);
        prefix = (prefix << 11) | bin;
    }
    __syncthreads();
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < a.old; i += (long long)gridDim.x * 256) {
        const uint32_t key = evict_key(a.total[i]);
        if (LEVEL == 2) { if ((key >> 21) == prefix) atomicAdd(&s_hist[(key >> 10) & 2047u], 1u); }
        else            { if ((key >> 10) == prefix) atomicAdd(&s_hist[key & 1023u], 1u); }
    }
    evict_flush(s_hist, a.hist + (LEVEL - 1) * GSR_EV_BINS, NB);
}

// The smallest key that stays, and how many rows with exactly that key do.
__device__ __forceinline__ void evict_threshold(const EvictArgs& a, uint32_t* s_tmp, uint32_t& key, uint32_t& ties)
{
    if (a.k == 0) { key = 0xffffffffu; ties = 0u; return; }                    // (no row has that key: +inf has 0xff800000)
    if (a.k == a.old) { key = 0u; ties = 0u; return; }                         // (nor this one: -inf has 0x007fffff)
    uint32_t b1, b2, b3, k;
    evict_pick(a.hist, GSR_EV_BINS / 256, (uint32_t)a.k, s_tmp, b1, k);
    evict_pick(a.hist + GSR_EV_BINS, GSR_EV_BINS / 256, k, s_tmp, b2, k);
    evict_pick(a.hist + 2 * GSR_EV_BINS, GSR_EV_BINS / 512, k, s_tmp, b3, ties);
    key = (b1 << 21) | (b2 << 10) | b3;
}

__global__ void __launch_bounds__(256) k_evict_count(EvictArgs a)
{
    __shared__ uint32_t s_tmp[8];
    __shared__ uint32_t s_n[2];
    uint32_t key, ties;
    evict_threshold(a, s_tmp, key, ties);
    if (threadIdx.x < 2) s_n[threadIdx.x] = 0u;
    __syncthreads();
    uint32_t above = 0, equal = 0;
    const long long lo = (long long)blockIdx.x * a.tile_rows;
    for (int r = threadIdx.x; r < a.tile_rows && lo + r < a.old; r += 256) {
        const uint32_t x = evict_key(a.total[lo + r]);
        above += x > key; equal += x == key;
    }
    atomicAdd(&s_n[0], above); atomicAdd(&s_n[1], equal);
    __syncthreads();
    if (threadIdx.x == 0) a.counts[blockIdx.x] = make_uint2(s_n[0], s_n[1]);
}

__global__ void __launch_bounds__(256) k_evict_emit(EvictArgs a)
{
    __shared__ uint32_t s_tmp[8];
    __shared__ uint32_t s_wave[4][2];
    __shared__ uint32_t s_base[2];
    uint32_t key, ties;
    evict_threshold(a, s_tmp, key, ties);
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    if (t < 2) s_base[t] = 0u;
    __syncthreads();
    uint32_t above = 0, equal = 0;          // of the tiles in front
    for (int b = t; b < (int)blockIdx.x; b += 256) { const uint2 n = a.counts[b]; above += n.x; equal += n.y; }
    atomicAdd(&s_base[0], above); atomicAdd(&s_base[1], equal);
    __syncthreads();
    above = s_base[0]; equal = s_base[1];
    const long long lo = (long long)blockIdx.x * a.tile_rows;
    for (int r0 = 0; r0 < a.tile_rows; r0 += 256) {          // (uniform: every thread meets the barriers)
        const long long i = lo + r0 + t;
        const bool in = r0 + t < a.tile_rows && i < a.P, recent = in && i >= a.old;
        const float s = in ? a.total[i] : 0.0f;
        const uint32_t x = in && !recent ? evict_key(s) : 0u;
        const bool is_above = in && !recent && x > key, is_equal = in && !recent && x == key;
        const unsigned long long ma = __ballot(is_above), me = __ballot(is_equal), below = (1ull << lane) - 1ull;
        if (lane == 0) { s_wave[wave][0] = (uint32_t)__popcll(ma); s_wave[wave][1] = (uint32_t)__popcll(me); }
        __syncthreads();
        uint32_t na = above, ne = equal, ta = 0, te = 0;
        for (int w = 0; w < 4; w++) {
            if (w < wave) { na += s_wave[w][0]; ne += s_wave[w][1]; }
            ta += s_wave[w][0]; te += s_wave[w][1];
        }
        na += (uint32_t)__popcll(ma & below); ne += (uint32_t)__popcll(me & below);
        long long at = -1;
        if (recent) at = (long long)a.k + (i - a.old);
        else if (is_above || (is_equal && ne < ties)) at = (long long)na + (ne < ties ? ne : ties);
        if (at >= 0) { a.kept[at] = i; a.scores_out[at] = s; }
        above += ta; equal += te;
        __syncthreads();
    }
}

struct RowTensor {
    const void* src; void* dst;
    const uint8_t* src_window; uint8_t* dst_window;          // codes of the 8-bit root: their windows (then a row's unit is one code)
    long long row;              // units of a row
    uint32_t first, pad;
    int unit;                   // bytes of a unit: 1, 2, 4, 8 or 16
};
struct RowArgs { int count; uint32_t chunks; long long keep; const long long* kept; RowTensor t[GSR_OPT_MAX]; };

template <class T>
__device__ __forceinline__ void evict_copy(const RowArgs& a, const RowTensor& t, uint32_t c)
{
    const long long base = (long long)(c - t.first) * GSR_OPT_CHUNK, n = a.keep * t.row;
    for (int k = threadIdx.x; k < GSR_OPT_CHUNK && base + k < n; k += GSR_OPT_THREADS) {
        const long long i = base + k, row = i / t.row;
        static_cast<T*>(t.dst)[i] = static_cast<const T*>(t.src)[a.kept[row] * t.row + (i - row * t.row)];
    }
}

// Codes change their block with their row: the float's upper bits move into the new block's window, exactly, but for what lies under
// that window (raised to its lowest value, as by the step).
__device__ __forceinline__ void evict_codes(const RowArgs& a, const RowTensor& t, uint32_t c)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint8_t* src = static_cast<const uint8_t*>(t.src);
    uint8_t* dst = static_cast<uint8_t*>(t.dst);
    const long long n = a.keep * t.row;
    for (int b = wave; b < GSR_OPT_CHUNK / GSR_OPT_WINDOW; b += 4) {
        const long long start = (long long)(c - t.first) * GSR_OPT_CHUNK + b * GSR_OPT_WINDOW;
        if (start >= n) break;
        uint32_t top[4], most = 0;
#pragma unroll
        for (int k = 0; k < 4; k++) {
            top[k] = 0;
            const long long i = start + 4 * lane + k;
            if (i < n) {
                const long long row = i / t.row, e = a.kept[row] * t.row + (i - row * t.row);
                const uint32_t code = src[e];
                if (code) top[k] = code + 16u * t.src_window[e / GSR_OPT_WINDOW] + 1u;
            }
            most = top[k] > most ? top[k] : most;
        }
        const uint32_t w = opt_window(wave_max_u32(most) << 19), now = 16u * w + 1u;
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const long long i = start + 4 * lane + k;
            if (i < n) dst[i] = top[k] == 0u ? 0 : (uint8_t)(top[k] > now + 1u ? top[k] - now : 1u);
        }
        if (lane == 0) t.dst_window[start / GSR_OPT_WINDOW] = (uint8_t)w;
    }
}

__global__ void __launch_bounds__(GSR_OPT_THREADS) k_evict_rows(RowArgs a)
{
    for (uint32_t c = blockIdx.x; c < a.chunks; c += gridDim.x) {
        const RowTensor& t = a.t[opt_find(a.t, a.count, c)];
        if (t.src_window) evict_codes(a, t, c);
        else if (t.unit == 16) evict_copy<uint4>(a, t, c);
        else if (t.unit == 8) evict_copy<uint2>(a, t, c);
        else if (t.unit == 4) evict_copy<uint32_t>(a, t, c);
        else if (t.unit == 2) evict_copy<uint16_t>(a, t, c);
        else evict_copy<uint8_t>(a, t, c);
    }
}

}  // namespace gsr
