// AdamW over many tensors at once, with the gradient's global norm and clipping.
//
// Mathematics (Loshchilov & Hutter, ICLR 2019), per element with g' = coef g:
//   m = b1 m + (1-b1) g';  v = b2 v + (1-b2) g'^2;  p = (1 - lr wd) p - lr / (1-b1^t) m / (sqrt(v) / sqrt(1-b2^t) + eps)
//   coef = grad_scale min(1, max_norm / (norm + 1e-6)),  norm = |grad_scale g| over ALL tensors
// The squares are summed in double: the product of two floats is exact there, so the norm, and with it coef, does not depend on the
// order of the sum in any bit that survives the rounding to float.
//
// Work split: the host cuts the tensors into chunks (a plan in device memory, made from the sizes alone) and a workgroup takes one
// chunk; the tensors' addresses travel in the kernel arguments, SS_ADAMW_PTRS tensors a launch (one launch for a flat buffer).
//
// Moments in 8 bits: a RUN of 256 elements shares one scale q per moment; a wave owns a run, four elements a lane, so the maximum of
// the run is six DPP steps in registers and nothing is staged.
//   first moment  = sign(c) c^2 q, |c| <= 127;   second moment = c^4 q, 0 <= c <= 255
// The power spaces the codes by about 2/c resp. 4/c of the value over four resp. nine decades, and its inverse is one resp. two square
// roots instead of a table.  Rounding is stochastic: b2 = 0.999 moves a second moment by far less than half a step, and rounding to
// nearest would hold it where it is for ever.  A positive second moment never takes code 0 (the update would divide by eps alone).
// The updated parameter uses the moments before they are rounded.
#include "common.h"
#include <cmath>

#define SS_ADAMW_PTRS 200
#define SS_ADAMW_GROUPS 64
#define SS_ADAMW_RUN 256

// 4 consecutive elements; addresses are aligned to the element only (a view may start anywhere), which global memory takes as one access
struct __attribute__((packed, aligned(4))) F4u { floatx4 v; };
struct __attribute__((packed, aligned(2))) H4u { bf16x4 v; };
__device__ __forceinline__ floatx4 load4(const float* p) { return ((const F4u*)p)->v; }
__device__ __forceinline__ floatx4 load4(const bf16* p) {
    const bf16x4 h = ((const H4u*)p)->v;
    floatx4 r;
#pragma unroll
    for (int e = 0; e < 4; ++e) r[e] = (float)h[e];
    return r;
}
__device__ __forceinline__ void store4(float* p, const floatx4& v) { ((F4u*)p)->v = v; }
__device__ __forceinline__ void store4(bf16* p, const floatx4& v) {
    bf16x4 h;
#pragma unroll
    for (int e = 0; e < 4; ++e) h[e] = (bf16)v[e];
    ((H4u*)p)->v = h;
}
// the first `n` (0..4) of four; the others read as zero and are not written
template <typename T> __device__ __forceinline__ floatx4 load_n(const T* p, int n) {
    if (n >= 4) return load4(p);
    floatx4 r = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int e = 0; e < 3; ++e) if (e < n) r[e] = to_f(p[e]);
    return r;
}
template <typename T> __device__ __forceinline__ void store_n(T* p, const floatx4& v, int n) {
    if (n >= 4) { store4(p, v); return; }
#pragma unroll
    for (int e = 0; e < 3; ++e) if (e < n) p[e] = from_f<T>(v[e]);
}

struct AdamChunk { int64_t start; int count, run, tensor, group; int64_t unused; };      // elements of a tensor; `run`: its first run in the state
static_assert(sizeof(AdamChunk) == 32, "the plan is built on the host as four 64-bit words a chunk");
struct AdamPtrs { const void* g[SS_ADAMW_PTRS]; };
struct AdamPtrs2 { void* p[SS_ADAMW_PTRS]; const void* g[SS_ADAMW_PTRS]; };

// What changes from step to step: by value, or made on the device by adamw_prepare_kernel
struct AdamDyn { float coef, rbc2; unsigned key; int skip; float step[SS_ADAMW_GROUPS], decay[SS_ADAMW_GROUPS]; };

__host__ __device__ __forceinline__ unsigned mix32(unsigned x) {       // odd multipliers: fractions of the golden ratio and of sqrt(3)
    x ^= x >> 16; x *= 0x9E3779B9u; x ^= x >> 15; x *= 0xBB67AE85u; return x ^ (x >> 16);
}
__host__ __device__ __forceinline__ unsigned step_key(unsigned seed, unsigned t) { return mix32(seed ^ mix32(t)); }

// ------------------------------------------------------------------ global norm: one partial sum (double) per workgroup
// A workgroup walks every gridDim-th chunk with a thread's eight vectors of a chunk in flight at once: with one workgroup a chunk the
// dependent loads before the first element (plan, address) are a third of its life.  81 M floats: 55 us = 5.8 TB/s alone, 84 - 103 us right
// behind kernels whose writes still drain.
#define SS_SQNORM_BLOCKS 1024
#define SS_ADAMW_JOIN_CHUNKS 4096
template <typename T>
__global__ __launch_bounds__(256) void multi_sqnorm_kernel(AdamPtrs ptrs, const AdamChunk* __restrict__ plan, int chunks, int first_tensor,
                                                           double* __restrict__ partial) {
    double s = 0.0;
    for (int k = blockIdx.x; k < chunks; k += gridDim.x) {
        const AdamChunk c = plan[k];
        const T* __restrict__ g = (const T*)ptrs.g[c.tensor - first_tensor];
        if (!g) continue;                                      // no gradient: nothing to add
        g += c.start;
        for (int o = threadIdx.x * 4; o < c.count; o += 8 * 1024) {
            floatx4 v[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) { const int e = o + u * 1024, n = c.count - e; v[u] = n > 0 ? load_n(g + e, n) : floatx4{0.f, 0.f, 0.f, 0.f}; }
#pragma unroll
            for (int u = 0; u < 8; ++u)
#pragma unroll
                for (int e = 0; e < 4; ++e) { const double d = (double)v[u][e]; s = fma(d, d, s); }
        }
    }
    __shared__ double sh[4];
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) partial[blockIdx.x] = (sh[0] + sh[1]) + (sh[2] + sh[3]);
}

struct AdamArgs {
    float b1, omb1, b2, omb2, eps;
    int sums;                                                  // partial sums of the norm, joined by every workgroup (small models)
    const double* partial;
    double max_norm, grad_scale;
    float* norm;
    AdamDyn dyn;
};

// Sum of up to a few thousand doubles by a workgroup of 256, in one order wherever it is taken
__device__ __forceinline__ double join_sums(const double* __restrict__ partial, int64_t count, double* sh) {
    double s = 0.0;
#pragma unroll 4
    for (int64_t i = threadIdx.x; i < count; i += 256) s += partial[i];
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = s;
    __syncthreads();
    return (sh[0] + sh[1]) + (sh[2] + sh[3]);
}
__device__ __forceinline__ float clip_coef(double norm, double max_norm, double grad_scale) {
    double clip = 1.0;
    if (max_norm > 0.0) { clip = max_norm / (norm + 1e-6); clip = clip > 1.0 ? 1.0 : clip; }        // NaN stays NaN
    return (float)(clip * grad_scale);
}
// What the gradients are multiplied by: made by adamw_prepare_kernel, joined here, or given
__device__ __forceinline__ float step_coef(const AdamArgs& a, const AdamDyn* __restrict__ dyn) {
    if (dyn) return dyn->coef;
    if (!a.partial) return a.dyn.coef;
    __shared__ double sh[4];
    const double norm = sqrt(join_sums(a.partial, a.sums, sh)) * fabs(a.grad_scale);
    if (a.norm && blockIdx.x == 0 && threadIdx.x == 0) *a.norm = (float)norm;
    return clip_coef(norm, a.max_norm, a.grad_scale);
}

// One workgroup: joins the partial sums in a fixed order, counts the step, and leaves what the update reads.  4.7 us, all latency, which is
// why small models join the sums in the update instead.
struct AdamSchedule { double lr[SS_ADAMW_GROUPS], wd[SS_ADAMW_GROUPS]; };
__global__ __launch_bounds__(256) void adamw_prepare_kernel(const double* __restrict__ partial, int64_t count, double max_norm, double grad_scale,
        double beta1, double beta2, int64_t t_host, int64_t* __restrict__ t_dev, AdamSchedule sched, const double* __restrict__ lr_dev, int groups,
        unsigned seed, int skip_nonfinite, float* __restrict__ norm_out, AdamDyn* __restrict__ dyn) {
    __shared__ double sh[4];
    __shared__ double bc1_s, bc2_s;
    __shared__ int64_t t_s;
    if (threadIdx.x == 64) {                                                // another wave than the one that ends the sum
        const int64_t t = t_dev ? *t_dev + 1 : t_host;                      // of a skipped step nothing is used
        t_s = t; bc1_s = 1.0 - pow(beta1, (double)t); bc2_s = 1.0 - pow(beta2, (double)t);
    }
    const double sum = join_sums(partial, count, sh);                       // its barrier also publishes what the other wave made
    if ((int)threadIdx.x < groups) {
        const double lr = lr_dev ? lr_dev[threadIdx.x] : sched.lr[threadIdx.x];
        dyn->step[threadIdx.x] = (float)(lr / bc1_s);
        dyn->decay[threadIdx.x] = (float)(1.0 - lr * sched.wd[threadIdx.x]);
    }
    if (threadIdx.x == 0) {
        const double norm = sqrt(sum) * fabs(grad_scale);
        const int skip = skip_nonfinite && !(norm < __builtin_huge_val());  // infinite or NaN
        if (t_dev && !skip) *t_dev = t_s;
        if (norm_out) *norm_out = (float)norm;
        dyn->coef = clip_coef(norm, max_norm, grad_scale); dyn->rbc2 = (float)(1.0 / sqrt(bc2_s)); dyn->key = step_key(seed, (unsigned)t_s); dyn->skip = skip;
    }
}

// ------------------------------------------------------------------ the update
__device__ __forceinline__ float adam_update(float p, float m, float v, float step, float decay, float rbc2, float eps) {
    const float denom = fmaf(__builtin_amdgcn_sqrtf(v), rbc2, eps);         // v_sqrt_f32 and v_rcp_f32: 1 ulp each of a term far below p
    return p * decay - step * m * __builtin_amdgcn_rcpf(denom);
}

// Products and sums of the moments are rounded one by one (no contraction): the code that a moment takes is a comparison, and the
// same operands give the same code whatever the compiler does.
__device__ __forceinline__ void adam_moments(float g, float& m, float& v, const AdamArgs& a) {
#pragma clang fp contract(off)
    const float mb = m * a.b1, mg = g * a.omb1;
    m = mb + mg;
    const float vb = v * a.b2, gg = g * g, vg = gg * a.omb2;
    v = vb + vg;
}

// 28 bytes an element in f32 (16 of them moments): 24 M elements 125 us = 5.4 TB/s, as fast as a copy.  Two vectors of each of the four
// streams in flight a thread; a chunk of at most 8192 elements, so that every workgroup is resident at once up to 16 M.
template <typename TP, typename TG>
__global__ __launch_bounds__(256) void adamw32_kernel(AdamPtrs2 ptrs, const AdamChunk* __restrict__ plan, int first_tensor, float* __restrict__ m,
        float* __restrict__ v, AdamArgs a, const AdamDyn* __restrict__ dyn) {
    if (dyn && dyn->skip) return;
    const AdamChunk c = plan[blockIdx.x];
    const float coef = step_coef(a, dyn), rbc2 = dyn ? dyn->rbc2 : a.dyn.rbc2;
    const float step = dyn ? dyn->step[c.group] : a.dyn.step[c.group], decay = dyn ? dyn->decay[c.group] : a.dyn.decay[c.group];
    const TG* __restrict__ g = (const TG*)ptrs.g[c.tensor - first_tensor];
    if (!g) return;                                            // no gradient: the tensor and its moments stay
    g += c.start;
    TP* __restrict__ p = (TP*)ptrs.p[c.tensor - first_tensor] + c.start;
    m += (int64_t)c.run * SS_ADAMW_RUN; v += (int64_t)c.run * SS_ADAMW_RUN;
    constexpr int U = 2;
    for (int o = threadIdx.x * 4; o < c.count; o += U * 1024) {
        floatx4 pv[U], gv[U], mv[U], vv[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int k = o + u * 1024, n = c.count - k;
            if (n > 0) { pv[u] = load_n(p + k, n); gv[u] = load_n(g + k, n); mv[u] = *(const floatx4*)(m + k); vv[u] = *(const floatx4*)(v + k); }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int k = o + u * 1024, n = c.count - k;
            if (n <= 0) continue;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                float mm = mv[u][e], vx = vv[u][e];
                adam_moments(gv[u][e] * coef, mm, vx, a);
                mv[u][e] = mm; vv[u][e] = vx;
                pv[u][e] = adam_update(pv[u][e], mm, vx, step, decay, rbc2, a.eps);
            }
            store_n(p + k, pv[u], n); *(floatx4*)(m + k) = mv[u]; *(floatx4*)(v + k) = vv[u];   // the state's slots are whole runs
        }
    }
}

// maximum over the 64 lanes of a wave, as unsigned bits: on |x| that is the order of the floats with NaN above infinity
template <int CTRL, int ROWS> __device__ __forceinline__ unsigned umax_dpp(unsigned v) {
    const unsigned o = (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xf, false);
    return v > o ? v : o;
}
__device__ __forceinline__ float wave_absmax(unsigned v) {
    v = umax_dpp<0xB1, 0xf>(v); v = umax_dpp<0x4E, 0xf>(v); v = umax_dpp<0x141, 0xf>(v); v = umax_dpp<0x140, 0xf>(v);
    v = umax_dpp<0x142, 0xa>(v); v = umax_dpp<0x143, 0xc>(v);              // row broadcasts: lane 63 ends with all four rows
    return __uint_as_float((unsigned)__builtin_amdgcn_readlane((int)v, 63));
}

__device__ __forceinline__ float grid_m(float c) { return c * c; }
__device__ __forceinline__ float grid_v(float c) { const float s = c * c; return s * s; }

// t in units of q -> the code below or above, above with probability (t - below) / (above - below); u16 = 0..65535.
// The square roots only guess: raised by 2^-22 (v_sqrt_f32 is good to 1 unit, two in a row to 1.5) the guess is the code below or one too
// high, and a comparison with the grid itself settles it, so the code does not depend on their rounding.
template <bool SECOND> __device__ __forceinline__ float encode(float t, float u16) {
#pragma clang fp contract(off)
    const float top = SECOND ? 254.f : 126.f;
    float c = __builtin_amdgcn_sqrtf(t);
    if (SECOND) c = __builtin_amdgcn_sqrtf(c);
    c = fminf(fmaxf(floorf(c * (1.f + 0x1p-22f)), 0.f), top);
    c = (SECOND ? grid_v(c) : grid_m(c)) > t ? c - 1.f : c;
    const float up = c + 1.f, below = SECOND ? grid_v(c) : grid_m(c), above = SECOND ? grid_v(up) : grid_m(up);
    const float gap = SECOND ? above - below : up + c, over = t - below, want = u16 * gap;
    c = over * 65536.f > want ? up : c;
    if (SECOND) c = fmaxf(c, t > 0.f ? 1.f : 0.f);
    return c;
}
__device__ __forceinline__ float decode_m(unsigned word, int e) {           // sign(c) c^2
    const float c = (float)((int)(word << (24 - 8 * e)) >> 24);
    return c * fabsf(c);
}

// 16 bytes an element and 1/16 in f32: 81 M elements 246 us = 5.3 TB/s; 3.3 M 18 us, 4.4 M of bf16 24 us.  447 vector instructions for four
// elements a lane, 34 of them at a quarter of the rate, take about as long as the bytes: more loads in flight (a resident grid with the
// next run on its way) cost more in registers than they gave (246 -> 270 us).
template <typename TP, typename TG>
__global__ __launch_bounds__(256) void adamw8_kernel(AdamPtrs2 ptrs, const AdamChunk* __restrict__ plan, int first_tensor, unsigned* __restrict__ mc,
        unsigned* __restrict__ vc, float* __restrict__ qm, float* __restrict__ qv, AdamArgs a, const AdamDyn* __restrict__ dyn) {
    if (dyn && dyn->skip) return;
    const AdamChunk c = plan[blockIdx.x];
    const float coef = step_coef(a, dyn), rbc2 = dyn ? dyn->rbc2 : a.dyn.rbc2;
    const float step = dyn ? dyn->step[c.group] : a.dyn.step[c.group], decay = dyn ? dyn->decay[c.group] : a.dyn.decay[c.group];
    const unsigned key = dyn ? dyn->key : a.dyn.key;
    const TG* __restrict__ g = (const TG*)ptrs.g[c.tensor - first_tensor];
    if (!g) return;                                            // no gradient: the tensor and its moments stay
    g += c.start;
    TP* __restrict__ p = (TP*)ptrs.p[c.tensor - first_tensor] + c.start;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int r = wave; r * SS_ADAMW_RUN < c.count; r += 4) {
        const int k = r * SS_ADAMW_RUN + lane * 4, n = c.count - k;
        const int run = c.run + r;
        const int64_t word = (int64_t)run * 64 + lane;
        floatx4 pv = {0.f, 0.f, 0.f, 0.f}, gv = pv;
        if (n > 0) { pv = load_n(p + k, n); gv = load_n(g + k, n); }
        const unsigned mw = mc[word], vw = vc[word];
        const float q1 = qm[run], q2 = qv[run];
        float m[4], v[4];
        unsigned mx = 0, vx = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            m[e] = decode_m(mw, e) * q1;
            v[e] = grid_v((float)((vw >> (8 * e)) & 255u)) * q2;
            adam_moments(gv[e] * coef, m[e], v[e], a);
            const unsigned bm = __float_as_uint(m[e]) & 0x7fffffffu, bv = __float_as_uint(v[e]) & 0x7fffffffu;
            mx = mx > bm ? mx : bm; vx = vx > bv ? vx : bv;
            pv[e] = adam_update(pv[e], m[e], v[e], step, decay, rbc2, a.eps);
        }
        if (n > 0) store_n(p + k, pv, n);
        const float bigm = wave_absmax(mx), bigv = wave_absmax(vx);
        // below 1e-28 a moment is held as zero (its scale and the scale's reciprocal stay normal floats); NaN stays NaN and marks the run
        const float s1 = bigm < 1e-28f ? 0.f : bigm * (float)(1.0 / 16129.0), s2 = bigv < 1e-28f ? 0.f : bigv * (float)(1.0 / (65025.0 * 65025.0));
        const float i1 = s1 > 0.f ? 1.f / s1 : 0.f, i2 = s2 > 0.f ? 1.f / s2 : 0.f;
        const unsigned rk = mix32(key + (unsigned)run * 0xBB67AE85u);
        unsigned mo = 0, vo = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const unsigned h = mix32(rk + (unsigned)(lane * 4 + e) * 0x9E3779B9u);
            const float cm = encode<false>(fabsf(m[e]) * i1, (float)(h & 0xffffu));
            const float cv = encode<true>(v[e] * i2, (float)(h >> 16));
            const int ci = (int)copysignf(cm, m[e]);
            mo |= ((unsigned)ci & 255u) << (8 * e);
            vo |= (unsigned)cv << (8 * e);
        }
        mc[word] = mo; vc[word] = vo;
        if (lane == 0) { qm[run] = s1; qv[run] = s2; }
    }
}

// the moments that 8-bit codes stand for: 2 bytes in, 8 out; 81 M elements 156 us = 5.2 TB/s
__global__ __launch_bounds__(256) void adamw8_values_kernel(const unsigned* __restrict__ mc, const unsigned* __restrict__ vc, const float* __restrict__ qm,
        const float* __restrict__ qv, float* __restrict__ m, float* __restrict__ v, int64_t words) {
    const int64_t stride = (int64_t)gridDim.x * 256;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < words; i += stride) {
        const unsigned mw = mc[i], vw = vc[i];
        const float q1 = qm[i >> 6], q2 = qv[i >> 6];
        floatx4 a, b;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            a[e] = decode_m(mw, e) * q1;
            b[e] = grid_v((float)((vw >> (8 * e)) & 255u)) * q2;
        }
        *(floatx4*)(m + i * 4) = a; *(floatx4*)(v + i * 4) = b;
    }
}

// ------------------------------------------------------------------ C ABI
static int check_list(const char* who, int count, const void* const* ptr, const int64_t* first_chunk, const void* plan, int64_t align, bool may_lack) {
    SS_CHECK(count >= 0 && (count == 0 || (ptr && first_chunk && first_chunk[0] == 0)), "%s: bad tensor list", who);
    for (int i = 0; i < count; ++i) {
        SS_CHECK(first_chunk[i + 1] >= first_chunk[i], "%s: chunk ranges must not fall (tensor %d)", who, i);
        SS_CHECK(first_chunk[i + 1] == first_chunk[i] || ((ptr[i] || may_lack) && (uintptr_t)ptr[i] % align == 0), "%s: tensor %d is null or misaligned", who, i);
    }
    SS_CHECK(count == 0 || first_chunk[count] < (1LL << 31), "%s: too many chunks", who);
    SS_CHECK(count == 0 || first_chunk[count] == 0 || plan, "%s: no plan", who);
    return 0;
}

static int64_t sqnorm_blocks(int64_t chunks) { return chunks < SS_SQNORM_BLOCKS ? chunks : SS_SQNORM_BLOCKS; }

extern "C" int64_t ss_multi_sqnorm_workspace(int count, const int64_t* first_chunk) {
    int64_t n = 0;
    for (int i0 = 0; first_chunk && i0 < count; i0 += SS_ADAMW_PTRS)
        n += sqnorm_blocks(first_chunk[count - i0 < SS_ADAMW_PTRS ? count : i0 + SS_ADAMW_PTRS] - first_chunk[i0]);
    return n * (int64_t)sizeof(double);
}

extern "C" int ss_multi_sqnorm(int dtype, int count, const void* const* grads, const int64_t* first_chunk, const void* plan, double* partial,
                               hipStream_t stream) {
    SS_CHECK(dtype == SS_F32 || dtype == SS_BF16, "ss_multi_sqnorm: unsupported dtype code %d", dtype);
    if (int rc = check_list("ss_multi_sqnorm", count, grads, first_chunk, plan, dtype == SS_F32 ? 4 : 2, true)) return rc;
    for (int i0 = 0; i0 < count; i0 += SS_ADAMW_PTRS) {
        const int n = count - i0 < SS_ADAMW_PTRS ? count - i0 : SS_ADAMW_PTRS;
        const int64_t c0 = first_chunk[i0], nc = first_chunk[i0 + n] - c0, blocks = sqnorm_blocks(nc);
        if (nc == 0) continue;
        SS_CHECK(partial, "ss_multi_sqnorm: no room for the partial sums");
        AdamPtrs t;
        memset(&t, 0, sizeof(t));
        for (int i = 0; i < n; ++i) t.g[i] = grads[i0 + i];
        SS_DISPATCH(dtype, hipLaunchKernelGGL((multi_sqnorm_kernel<T>), dim3((unsigned)blocks), dim3(256), 0, stream, t, (const AdamChunk*)plan + c0, (int)nc,
                                              i0, partial));
        SS_LAUNCH_CHECK();
        partial += blocks;
    }
    return 0;
}

extern "C" int64_t ss_adamw_dyn_workspace(void) { return (int64_t)sizeof(AdamDyn); }

static int check_hyper(const char* who, int groups, const double* lr, const double* wd, double beta1, double beta2, double grad_scale) {
    SS_CHECK(groups > 0 && groups <= SS_ADAMW_GROUPS && lr && wd, "%s: 1 to %d parameter groups, got %d", who, SS_ADAMW_GROUPS, groups);
    SS_CHECK(beta1 >= 0.0 && beta1 < 1.0 && beta2 >= 0.0 && beta2 < 1.0, "%s: betas must lie in [0, 1)", who);
    SS_CHECK(std::isfinite(grad_scale), "%s: grad_scale must be finite", who);
    return 0;
}

extern "C" int ss_adamw_prepare(const double* partial, int64_t count, double max_norm, double grad_scale, double beta1, double beta2, int64_t t,
                                int64_t* t_dev, int groups, const double* lr, const double* weight_decay, const double* lr_dev, int64_t seed,
                                int skip_nonfinite, float* norm, void* dyn, hipStream_t stream) {
    if (int rc = check_hyper("ss_adamw_prepare", groups, lr, weight_decay, beta1, beta2, grad_scale)) return rc;
    SS_CHECK(dyn && count >= 0 && (count == 0 || partial) && (t_dev || t >= 1), "ss_adamw_prepare: bad arguments");
    AdamSchedule s;
    memset(&s, 0, sizeof(s));
    for (int i = 0; i < groups; ++i) { s.lr[i] = lr[i]; s.wd[i] = weight_decay[i]; }
    hipLaunchKernelGGL(adamw_prepare_kernel, dim3(1), dim3(256), 0, stream, partial, count, max_norm, grad_scale, beta1, beta2, t, t_dev, s, lr_dev,
                       groups, (unsigned)seed, skip_nonfinite, norm, (AdamDyn*)dyn);
    SS_LAUNCH_CHECK();
    return 0;
}

struct AdamNorm { const double* partial; int sums; double max_norm; float* norm; };
static int adamw_step(int p_dtype, int g_dtype, int bits, int count, void* const* params, const void* const* grads, const int64_t* first_chunk,
                             const void* plan, void* m, void* v, float* m_scale, float* v_scale, double beta1, double beta2, double eps,
                             double grad_scale, int64_t t, int groups, const double* lr, const double* weight_decay, int64_t seed, const void* dyn,
                      const AdamNorm& joined, hipStream_t stream) {
    SS_CHECK((p_dtype == SS_F32 || p_dtype == SS_BF16) && (g_dtype == SS_F32 || g_dtype == SS_BF16), "ss_adamw_step: unsupported dtype codes %d / %d", p_dtype, g_dtype);
    SS_CHECK(bits == 32 || bits == 8, "ss_adamw_step: moments of 32 or 8 bits, got %d", bits);
    if (int rc = check_hyper("ss_adamw_step", groups, lr, weight_decay, beta1, beta2, grad_scale)) return rc;
    if (int rc = check_list("ss_adamw_step", count, (const void* const*)params, first_chunk, plan, p_dtype == SS_F32 ? 4 : 2, false)) return rc;
    if (int rc = check_list("ss_adamw_step", count, grads, first_chunk, plan, g_dtype == SS_F32 ? 4 : 2, true)) return rc;
    SS_CHECK(eps >= 0.0 && (dyn || t >= 1), "ss_adamw_step: eps >= 0 and a step count from 1 on");
    if (count == 0 || first_chunk[count] == 0) return 0;
    SS_CHECK(m && v && aligned16(m) && aligned16(v) && (bits == 32 || (m_scale && v_scale)), "ss_adamw_step: state is missing or not 16-byte aligned");
    AdamArgs a;
    memset(&a, 0, sizeof(a));
    a.b1 = (float)beta1; a.omb1 = (float)(1.0 - beta1); a.b2 = (float)beta2; a.omb2 = (float)(1.0 - beta2); a.eps = (float)eps;   // each rounded once
    a.partial = joined.partial; a.sums = joined.sums; a.max_norm = joined.max_norm; a.grad_scale = grad_scale; a.norm = joined.norm;
    if (!dyn) {
        const double bc1 = 1.0 - pow(beta1, (double)t), bc2 = 1.0 - pow(beta2, (double)t);
        a.dyn.coef = (float)grad_scale; a.dyn.rbc2 = (float)(1.0 / sqrt(bc2)); a.dyn.key = step_key((unsigned)seed, (unsigned)t);
        for (int i = 0; i < groups; ++i) { a.dyn.step[i] = (float)(lr[i] / bc1); a.dyn.decay[i] = (float)(1.0 - lr[i] * weight_decay[i]); }
    }
    constexpr int PER = SS_ADAMW_PTRS;
    for (int i0 = 0; i0 < count; i0 += PER) {
        const int n = count - i0 < PER ? count - i0 : PER;
        const int64_t c0 = first_chunk[i0], nc = first_chunk[i0 + n] - c0;
        if (nc == 0) continue;
        AdamPtrs2 ptr;
        memset(&ptr, 0, sizeof(ptr));
        for (int i = 0; i < n; ++i) { ptr.p[i] = params[i0 + i]; ptr.g[i] = grads[i0 + i]; }
        const AdamChunk* pl = (const AdamChunk*)plan + c0;
#define SS_ADAMW(TP, TG) do { \
        if (bits == 32) hipLaunchKernelGGL((adamw32_kernel<TP, TG>), dim3((unsigned)nc), dim3(256), 0, stream, ptr, pl, i0, (float*)m, (float*)v, a, (const AdamDyn*)dyn); \
        else hipLaunchKernelGGL((adamw8_kernel<TP, TG>), dim3((unsigned)nc), dim3(256), 0, stream, ptr, pl, i0, (unsigned*)m, (unsigned*)v, m_scale, v_scale, a, (const AdamDyn*)dyn); } while (0)
        if (p_dtype == SS_F32) { if (g_dtype == SS_F32) SS_ADAMW(float, float); else SS_ADAMW(float, bf16); }
        else { if (g_dtype == SS_F32) SS_ADAMW(bf16, float); else SS_ADAMW(bf16, bf16); }
#undef SS_ADAMW
        SS_LAUNCH_CHECK();
        a.norm = nullptr;                                      // the first launch has written it
    }
    return 0;
}

extern "C" int ss_adamw_step(int p_dtype, int g_dtype, int bits, int count, void* const* params, const void* const* grads, const int64_t* first_chunk,
                             const void* plan, void* m, void* v, float* m_scale, float* v_scale, double beta1, double beta2, double eps,
                             double grad_scale, int64_t t, int groups, const double* lr, const double* weight_decay, int64_t seed, const void* dyn,
                             hipStream_t stream) {
    return adamw_step(p_dtype, g_dtype, bits, count, params, grads, first_chunk, plan, m, v, m_scale, v_scale, beta1, beta2, eps, grad_scale, t, groups, lr,
                      weight_decay, seed, dyn, AdamNorm{nullptr, 0, 0.0, nullptr}, stream);
}

// norm, preparation and update behind one call: a small model's step is the host's time
extern "C" int ss_adamw_clip_step(int p_dtype, int g_dtype, int bits, int count, void* const* params, const void* const* grads, const int64_t* first_chunk,
                                  const void* plan, void* m, void* v, float* m_scale, float* v_scale, double beta1, double beta2, double eps,
                                  double grad_scale, int64_t t, int groups, const double* lr, const double* weight_decay, int64_t seed, double max_norm,
                                  int skip_nonfinite, int64_t* t_dev, const double* lr_dev, float* norm, void* dyn, double* partial, hipStream_t stream) {
    SS_CHECK(dyn, "ss_adamw_clip_step: no room for the step's scalars");
    int64_t sums = 0;
    if (partial) {
        if (int rc = ss_multi_sqnorm(g_dtype, count, grads, first_chunk, plan, partial, stream)) return rc;
        sums = ss_multi_sqnorm_workspace(count, first_chunk) / (int64_t)sizeof(double);
    }
    // few chunks: every workgroup joins the partial sums itself, which saves a launch of 4 us; many would read them too often
    if (partial && !t_dev && !lr_dev && !skip_nonfinite && count > 0 && first_chunk[count] > 0 && first_chunk[count] <= SS_ADAMW_JOIN_CHUNKS) {
        SS_CHECK(max_norm > 0.0 || norm, "ss_adamw_clip_step: a norm that nobody asked for");
        return adamw_step(p_dtype, g_dtype, bits, count, params, grads, first_chunk, plan, m, v, m_scale, v_scale, beta1, beta2, eps, grad_scale, t, groups,
                          lr, weight_decay, seed, nullptr, AdamNorm{partial, (int)sums, max_norm, norm}, stream);
    }
    if (int rc = ss_adamw_prepare(partial, sums, max_norm, grad_scale, beta1, beta2, t, t_dev, groups, lr, weight_decay, lr_dev, seed, skip_nonfinite, norm,
                                  dyn, stream)) return rc;
    return ss_adamw_step(p_dtype, g_dtype, bits, count, params, grads, first_chunk, plan, m, v, m_scale, v_scale, beta1, beta2, eps, grad_scale, t, groups, lr,
                         weight_decay, seed, dyn, stream);
}

extern "C" int ss_adamw8_values(const void* m, const void* v, const float* m_scale, const float* v_scale, float* m_out, float* v_out, int64_t runs,
                                hipStream_t stream) {
    SS_CHECK(runs >= 0, "ss_adamw8_values: runs < 0");
    if (runs == 0) return 0;
    SS_CHECK(m && v && m_scale && v_scale && m_out && v_out && aligned16(m) && aligned16(v) && aligned16(m_out) && aligned16(v_out),
             "ss_adamw8_values: missing or misaligned buffers");
    const int64_t words = runs * 64, blocks = cdiv(words, 256);
    hipLaunchKernelGGL(adamw8_values_kernel, dim3((unsigned)(blocks < 8192 ? blocks : 8192)), dim3(256), 0, stream, (const unsigned*)m, (const unsigned*)v,
                       m_scale, v_scale, m_out, v_out, words);
    SS_LAUNCH_CHECK();
    return 0;
}
