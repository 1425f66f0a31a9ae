// srgen_optim_kernels.hip -- optimizer operators over a list of tensors: AdamW with moments in 32 or 8 bits, the total
// gradient norm, scaling in place, and moments written to / read from 8 bits.
#include "srgen_optim.h"

namespace srgen {
namespace {

// unaligned vectors: a gradient that is a view into a flat buffer starts at any element (global loads need element alignment only)
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));
typedef unsigned short u16x4u __attribute__((ext_vector_type(4), aligned(2)));

constexpr uint32_t kGold = 0x9E3779B9u;        // 2^32 / golden ratio: consecutive steps and high words get far keys

__host__ __device__ inline uint32_t mix32(uint32_t x)
{
    x ^= x >> 16;
    x *= 0x5340508Du;
    x ^= x >> 15;
    x *= 0x7495C5A5u;
    return x ^ (x >> 16);
}

__device__ inline float bf16_to_f32(uint32_t h) { return __uint_as_float(h << 16); }

template <int DT>                              // 0 fp32, 1 bf16, 2 fp16
__device__ inline void load_quad(const void* base, uint64_t i, uint64_t n, float (&x)[4])
{
    if constexpr (DT == 0) {
        const float* q = (const float*)base + i;
        if (i + 4 <= n) {
            const f32x4u a = *(const f32x4u*)q;
#pragma unroll
            for (int k = 0; k < 4; ++k) x[k] = a[k];
        } else {
#pragma unroll
            for (int k = 0; k < 4; ++k) x[k] = i + k < n ? q[k] : 0.f;
        }
    } else {
        const unsigned short* q = (const unsigned short*)base + i;
        unsigned short h[4];
        if (i + 4 <= n) {
            const u16x4u a = *(const u16x4u*)q;
#pragma unroll
            for (int k = 0; k < 4; ++k) h[k] = a[k];
        } else {
#pragma unroll
            for (int k = 0; k < 4; ++k) h[k] = i + k < n ? q[k] : (unsigned short)0;
        }
#pragma unroll
        for (int k = 0; k < 4; ++k)
            x[k] = DT == 1 ? bf16_to_f32(h[k]) : (float)__builtin_bit_cast(_Float16, h[k]);
    }
}

__device__ inline void load_quad_dt(int dt, const void* base, uint64_t i, uint64_t n, float (&x)[4])
{
    if (dt == 0) load_quad<0>(base, i, n, x);
    else if (dt == 1) load_quad<1>(base, i, n, x);
    else load_quad<2>(base, i, n, x);
}

__device__ inline void store_f32(float* q, uint64_t i, uint64_t n, const float (&x)[4])
{
    q += i;
    if (i + 4 <= n) {
        f32x4u a;
#pragma unroll
        for (int k = 0; k < 4; ++k) a[k] = x[k];
        *(f32x4u*)q = a;
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (i + k < n) q[k] = x[k];
    }
}

__device__ inline void store_u16(unsigned short* q, uint64_t i, uint64_t n, const unsigned short (&x)[4])
{
    q += i;
    if (i + 4 <= n) {
        u16x4u a;
#pragma unroll
        for (int k = 0; k < 4; ++k) a[k] = x[k];
        *(u16x4u*)q = a;
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (i + k < n) q[k] = x[k];
    }
}

// bf16 by stochastic rounding: 16 random bits under the last kept one, the rest cut off
__device__ inline unsigned short bf16_stochastic(float x, uint32_t rnd16)
{
    const uint32_t b = __float_as_uint(x);
    if ((b & 0x7F800000u) == 0x7F800000u) return (unsigned short)((b >> 16) | ((b & 0x7FFFFFu) ? 0x40u : 0u));
    return (unsigned short)((b + rnd16) >> 16);
}

__device__ inline unsigned short bf16_nearest(float x)
{
    const uint32_t b = __float_as_uint(x);
    if ((b & 0x7F800000u) == 0x7F800000u) return (unsigned short)((b >> 16) | ((b & 0x7FFFFFu) ? 0x40u : 0u));
    return (unsigned short)((b + 0x7FFFu + ((b >> 16) & 1u)) >> 16);
}

// ---- e4m3 with a power of two for each block of 32 ---------------------------------------------------------------------
// The scale 2^(e - 127) puts the block's largest magnitude at 2^8 .. 1.75 * 2^8, e4m3's top (a magnitude of 1.75 * 2^k to
// 2^(k+1) goes one binade down, so that rounding up cannot pass the top).  Not finite counts as 0 here and is stored as NaN.
__device__ inline uint32_t finite_bits(float x)
{
    const uint32_t b = __float_as_uint(x) & 0x7FFFFFFFu;
    return b >= 0x7F800000u ? 0u : b;
}

constexpr uint32_t kTop = 0x7F600000u;         // 1.75 * 2^127: what is above is stored as it, or it would round up to infinity

__device__ inline uint32_t scale_byte(uint32_t top_bits)
{
    top_bits = top_bits < kTop ? top_bits : kTop;
    const uint32_t e = (top_bits + 0x1FFFFFu) >> 23;
    return (e < 9u ? 9u : e) - 8u;
}

__device__ inline uint32_t e4m3_code(float x, uint32_t e, uint32_t rnd16, bool positive)
{
    const uint32_t b = __float_as_uint(x), mag = b & 0x7FFFFFFFu;
    const float y = __uint_as_float(mag < kTop ? mag : kTop) * __uint_as_float((254u - e) << 23);        // |x| / 2^(e - 127), exact where it matters
    const uint32_t normal = ((__float_as_uint(y) + (rnd16 << 4)) >> 20) - 960u;      // e4m3's exponent bias is 7: 960 = (127 - 7) * 8
    const uint32_t small = ((uint32_t)(y * 33554432.f) + rnd16) >> 16;               // below 2^-6: multiples of 2^-9
    uint32_t c = y < 0.015625f ? small : normal;
    if (positive && c == 0u && mag != 0u) c = 1u;
    if (mag >= 0x7F800000u) c = 0x7Fu;
    return c | ((b >> 24) & 0x80u);
}

__device__ inline float e4m3_value(uint32_t c)               // in units of the block's scale
{
    return __builtin_amdgcn_cvt_f32_fp8((int)c, 0);
}

// the power of two a scale byte stands for (e8m0: 0 is 2^-127, 255 NaN)
__device__ inline float scale_value(uint32_t e)
{
    return __uint_as_float(e == 0u ? 0x00400000u : e == 255u ? 0x7FC00000u : e << 23);
}

__device__ inline uint32_t max8(uint32_t x)                  // over the 8 lanes that hold one block
{
#pragma unroll
    for (int d = 1; d < 8; d <<= 1) {
        const uint32_t o = (uint32_t)__shfl_xor((int)x, d);
        x = x > o ? x : o;
    }
    return x;
}

// which tensor of the launch a workgroup works on: the last one with block0 <= blk
__device__ inline int find_tensor(const OptTensors& ts, uint32_t blk)
{
    int lo = 0, hi = ts.count - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (ts.t[mid].block0 <= blk) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

// ---- AdamW -------------------------------------------------------------------------------------------------------------
//   g' = c g      m = b1 m + (1 - b1) g'      v = b2 v + (1 - b2) g'^2
//   p  = (1 - lr wd) p - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
// One workgroup owns kOptChunk consecutive elements of one tensor and that chunk's step counter, so t needs no second launch
// and no atomics: every chunk of a tensor counts the same steps.
template <int BITS>
__global__ __launch_bounds__(256) void adamw_many_kernel(const AdamWArgs a)
{
    const AdamWScalars& sc = a.sc;
    const int ti = find_tensor(a.ts, blockIdx.x);
    const OptTensor& T = a.ts.t[ti];
    if (T.g == nullptr) return;
    if (sc.found_inf && *sc.found_inf != 0.f) return;
    const uint64_t n = T.numel_flags & kNumelMask;
    const int pdt = (int)(T.numel_flags >> 48) & 15, gdt = (int)(T.numel_flags >> 52) & 15;
    const uint64_t base = (uint64_t)(blockIdx.x - T.block0) * kOptChunk;
    const uint64_t off = (uint64_t)T.offset32 * kOptBlock;
    int32_t* counter = a.mo.step + (size_t)a.ts.counter0 + blockIdx.x;
    const int t = *counter + 1;
    __syncthreads();                                        // every wave has read the counter
    if (threadIdx.x == 0) *counter = t;

    const double lr = sc.lr_dev ? (double)*sc.lr_dev : sc.lr;
    const double bc1 = -expm1((double)t * sc.ln_beta1), bc2 = -expm1((double)t * sc.ln_beta2);
    const float decay = (float)(1.0 - lr * sc.wd), step = (float)(lr / bc1), isb2 = (float)(1.0 / sqrt(bc2)), eps = (float)sc.eps;
    double gmul = sc.grad_mul ? (double)*sc.grad_mul : 1.0;
    if (sc.grad_div) gmul /= (double)*sc.grad_div;
    if (sc.negate) gmul = -gmul;
    const uint32_t key = mix32(sc.seed_key + (uint32_t)t * kGold);

    for (int it = 0; it < kOptChunk / 1024; ++it) {
        const uint64_t i = base + it * 1024 + threadIdx.x * 4;
        if (i >= ((n + kOptBlock - 1) & ~(uint64_t)(kOptBlock - 1))) break;            // (whole blocks of 32: 8 lanes)
        const uint64_t j = off + i;
        float p[4], g[4], m[4], r[4];
        load_quad_dt(pdt, T.p, i, n, p);
        load_quad_dt(gdt, T.g, i, n, g);
        uint32_t h[4];
        if (BITS == 8 || pdt == 1) {
            const uint32_t hi = (uint32_t)(j >> 32) * kGold;
#pragma unroll
            for (int k = 0; k < 4; ++k) h[k] = mix32(((uint32_t)j + k + hi) ^ key);
        }
        if constexpr (BITS == 32) {
            float* mp = (float*)a.mo.m + j;
            float* vp = (float*)a.mo.v + j;
            float4 m4 = *(const float4*)mp, v4 = *(const float4*)vp;
            const float b1 = (float)sc.beta1, c1 = (float)(1.0 - sc.beta1), b2 = (float)sc.beta2, c2 = (float)(1.0 - sc.beta2);
            const float gm = (float)gmul;
            float* mq = (float*)&m4;
            float* vq = (float*)&v4;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float gk = g[k] * gm;
                mq[k] = fmaf(b1, mq[k], c1 * gk);
                vq[k] = fmaf(b2, vq[k], (c2 * gk) * gk);
                m[k] = mq[k];
                r[k] = sqrtf(vq[k]);
            }
            *(float4*)mp = m4;
            *(float4*)vp = v4;
        } else {
            uint8_t* mp = (uint8_t*)a.mo.m + j;
            uint8_t* vp = (uint8_t*)a.mo.v + j;
            uint8_t* mep = a.mo.m_scale + j / kOptBlock;
            uint8_t* vep = a.mo.v_scale + j / kOptBlock;
            const uint32_t mc = *(const uint32_t*)mp, vc = *(const uint32_t*)vp;
            const float ms = scale_value(*mep), vs = scale_value(*vep);
            uint32_t mt = 0, rt = 0;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const double gk = (double)g[k] * gmul;
                const float mo = e4m3_value((mc >> (8 * k)) & 255u) * ms, ro = e4m3_value((vc >> (8 * k)) & 255u) * vs;
                m[k] = (float)(sc.beta1 * (double)mo + (1.0 - sc.beta1) * gk);
                const float v = (float)(sc.beta2 * ((double)ro * (double)ro) + (1.0 - sc.beta2) * (gk * gk));
                r[k] = sqrtf(v);
                const uint32_t mb = finite_bits(m[k]), rb = finite_bits(r[k]);
                mt = mt > mb ? mt : mb;
                rt = rt > rb ? rt : rb;
            }
            const uint32_t me = scale_byte(max8(mt)), re = scale_byte(max8(rt));
            uint32_t mn = 0, rn = 0;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                mn |= e4m3_code(m[k], me, h[k] & 0xFFFFu, false) << (8 * k);
                rn |= e4m3_code(r[k], re, h[k] >> 16, true) << (8 * k);
            }
            *(uint32_t*)mp = mn;
            *(uint32_t*)vp = rn;
            if ((threadIdx.x & 7) == 0) {
                *mep = (uint8_t)me;
                *vep = (uint8_t)re;
            }
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) p[k] = fmaf(p[k], decay, -step * (m[k] / fmaf(r[k], isb2, eps)));
        if (pdt == 0) store_f32((float*)T.p, i, n, p);
        else {
            unsigned short q[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) q[k] = bf16_stochastic(p[k], mix32(h[k] + kGold) >> 16);
            store_u16((unsigned short*)T.p, i, n, q);
        }
    }
}

// ---- total norm --------------------------------------------------------------------------------------------------------
__device__ inline double wave_sum(double x)
{
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) x += __shfl_xor(x, d);
    return x;
}

// sums of squares in 64 bits, in a fixed order: one partial sum for each workgroup's elements
__global__ __launch_bounds__(256) void norm_partial_kernel(const OptTensors ts, uint32_t per_block, double* __restrict__ partial)
{
    __shared__ double red[4];
    const int ti = find_tensor(ts, blockIdx.x);
    const OptTensor& T = ts.t[ti];
    const uint64_t n = T.numel_flags & kNumelMask;
    const int dt = (int)(T.numel_flags >> 48) & 15;
    const uint64_t base = (uint64_t)(blockIdx.x - T.block0) * per_block;
    const uint64_t end = base + per_block < n ? base + per_block : n;
    double acc = 0.0;
    for (uint64_t i = base + threadIdx.x * 4; i < end; i += 1024) {
        float g[4];
        load_quad_dt(dt, T.g, i, n, g);
#pragma unroll
        for (int k = 0; k < 4; ++k) acc = fma((double)g[k], (double)g[k], acc);
    }
    acc = wave_sum(acc);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = acc;
    __syncthreads();
    if (threadIdx.x == 0) partial[(size_t)ts.counter0 + blockIdx.x] = (red[0] + red[1]) + (red[2] + red[3]);
}

// norm_coef[0] = sqrt(sum), norm_coef[1] = min(1, max_norm / (norm + 1e-6)); a NaN norm gives a NaN coefficient
__global__ __launch_bounds__(1024) void norm_final_kernel(const double* __restrict__ partial, uint32_t n, double max_norm,
                                                          float* __restrict__ norm_coef)
{
    __shared__ double red[16];
    double acc = 0.0;
    for (uint32_t i = threadIdx.x; i < n; i += 1024) acc += partial[i];
    acc = wave_sum(acc);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = acc;
    __syncthreads();
    if (threadIdx.x == 0) {
        double s = 0.0;
#pragma unroll
        for (int k = 0; k < 16; ++k) s += red[k];
        const float norm = (float)sqrt(s);
        const double c = max_norm / ((double)norm + 1e-6);
        norm_coef[0] = norm;
        norm_coef[1] = c > 1.0 ? 1.f : (float)c;
    }
}

// g *= *coef, rounded to nearest; a coefficient of 1 leaves the tensors alone
__global__ __launch_bounds__(256) void scale_many_kernel(const OptTensors ts, const float* __restrict__ coef)
{
    const float c = *coef;
    if (c == 1.f) return;
    const int ti = find_tensor(ts, blockIdx.x);
    const OptTensor& T = ts.t[ti];
    const uint64_t n = T.numel_flags & kNumelMask;
    const int dt = (int)(T.numel_flags >> 48) & 15;
    const uint64_t base = (uint64_t)(blockIdx.x - T.block0) * kOptChunk;
    for (int it = 0; it < kOptChunk / 1024; ++it) {
        const uint64_t i = base + it * 1024 + threadIdx.x * 4;
        if (i >= n) break;
        float g[4];
        load_quad_dt(dt, T.p, i, n, g);
#pragma unroll
        for (int k = 0; k < 4; ++k) g[k] *= c;
        if (dt == 0) store_f32((float*)T.p, i, n, g);
        else {
            unsigned short q[4];
#pragma unroll
            for (int k = 0; k < 4; ++k)
                q[k] = dt == 1 ? bf16_nearest(g[k]) : __builtin_bit_cast(unsigned short, (_Float16)g[k]);
            store_u16((unsigned short*)T.p, i, n, q);
        }
    }
}

// ---- moments to 8 bits and back ----------------------------------------------------------------------------------------
// to the nearest: the stochastic rounding's cut with half a step added; values that 8 bits hold come back as they are
__global__ __launch_bounds__(256) void moments_pack_kernel(const float* __restrict__ m, const float* __restrict__ v, uint64_t n,
                                                           uint8_t* __restrict__ m8, uint8_t* __restrict__ me, uint8_t* __restrict__ r8,
                                                           uint8_t* __restrict__ re)
{
    const uint64_t i = ((uint64_t)blockIdx.x * 256 + threadIdx.x) * 4;
    if (i >= ((n + kOptBlock - 1) & ~(uint64_t)(kOptBlock - 1))) return;
    float a[4], b[4];
    load_quad<0>(m, i, n, a);
    load_quad<0>(v, i, n, b);
    uint32_t mt = 0, rt = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        b[k] = sqrtf(b[k]);
        const uint32_t mb = finite_bits(a[k]), rb = finite_bits(b[k]);
        mt = mt > mb ? mt : mb;
        rt = rt > rb ? rt : rb;
    }
    const uint32_t em = scale_byte(max8(mt)), er = scale_byte(max8(rt));
    uint32_t mn = 0, rn = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        mn |= e4m3_code(a[k], em, 0x8000u, false) << (8 * k);
        rn |= e4m3_code(b[k], er, 0x8000u, true) << (8 * k);
    }
    *(uint32_t*)(m8 + i) = mn;
    *(uint32_t*)(r8 + i) = rn;
    if ((threadIdx.x & 7) == 0) {
        me[i / kOptBlock] = (uint8_t)em;
        re[i / kOptBlock] = (uint8_t)er;
    }
}

__global__ __launch_bounds__(256) void moments_unpack_kernel(const uint8_t* __restrict__ m8, const uint8_t* __restrict__ me,
                                                             const uint8_t* __restrict__ r8, const uint8_t* __restrict__ re,
                                                             float* __restrict__ m, float* __restrict__ v, uint64_t n)
{
    const uint64_t i = ((uint64_t)blockIdx.x * 256 + threadIdx.x) * 4;
    if (i >= n) return;
    const uint32_t mc = *(const uint32_t*)(m8 + i), rc = *(const uint32_t*)(r8 + i);
    const float ms = scale_value(me[i / kOptBlock]), rs = scale_value(re[i / kOptBlock]);
    float a[4], b[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        a[k] = e4m3_value((mc >> (8 * k)) & 255u) * ms;
        const float x = e4m3_value((rc >> (8 * k)) & 255u) * rs;
        b[k] = x * x;
    }
    store_f32(m, i, n, a);
    store_f32(v, i, n, b);
}

}  // namespace

uint32_t opt_mix(uint32_t x) { return mix32(x); }

hipError_t launch_adamw_many(const AdamWArgs& a, int bits, uint32_t blocks, hipStream_t s)
{
    if (bits == 32) hipLaunchKernelGGL(adamw_many_kernel<32>, dim3(blocks), dim3(256), 0, s, a);
    else hipLaunchKernelGGL(adamw_many_kernel<8>, dim3(blocks), dim3(256), 0, s, a);
    return hipGetLastError();
}

hipError_t launch_norm_partial(const OptTensors& ts, uint32_t blocks, uint32_t per_block, double* partial, hipStream_t s)
{
    hipLaunchKernelGGL(norm_partial_kernel, dim3(blocks), dim3(256), 0, s, ts, per_block, partial);
    return hipGetLastError();
}

hipError_t launch_norm_final(const double* partial, uint32_t n, double max_norm, float* norm_coef, hipStream_t s)
{
    hipLaunchKernelGGL(norm_final_kernel, dim3(1), dim3(1024), 0, s, partial, n, max_norm, norm_coef);
    return hipGetLastError();
}

hipError_t launch_scale_many(const OptTensors& ts, uint32_t blocks, const float* coef, hipStream_t s)
{
    hipLaunchKernelGGL(scale_many_kernel, dim3(blocks), dim3(256), 0, s, ts, coef);
    return hipGetLastError();
}

hipError_t launch_moments_pack(const float* m, const float* v, size_t n, uint8_t* m8, uint8_t* me, uint8_t* r8, uint8_t* re,
                               hipStream_t s)
{
    const uint64_t quads = ((n + kOptBlock - 1) / kOptBlock) * (kOptBlock / 4);
    hipLaunchKernelGGL(moments_pack_kernel, dim3((unsigned)((quads + 255) / 256)), dim3(256), 0, s, m, v, (uint64_t)n, m8, me, r8, re);
    return hipGetLastError();
}

hipError_t launch_moments_unpack(const uint8_t* m8, const uint8_t* me, const uint8_t* r8, const uint8_t* re, float* m, float* v,
                                 size_t n, hipStream_t s)
{
    const uint64_t quads = (n + 3) / 4;
    hipLaunchKernelGGL(moments_unpack_kernel, dim3((unsigned)((quads + 255) / 256)), dim3(256), 0, s, m8, me, r8, re, m, v, (uint64_t)n);
    return hipGetLastError();
}

}  // namespace srgen
