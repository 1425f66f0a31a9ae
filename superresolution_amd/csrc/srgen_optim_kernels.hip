// srgen_optim_kernels.hip -- optimizer operators over a list of tensors: AdamW with moments in 32 or 8 bits, the total
// gradient norm, scaling in place, and moments written to / read from 8 bits.
#include "srgen_optim.h"

namespace srgen {
namespace {

// unaligned vectors: a gradient that is a view into a flat buffer starts at any element (global loads need element alignment only)
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));
typedef unsigned short u16x4u __attribute__((ext_vector_type(4), aligned(2)));
// an address that came as a number is in device memory: without this it would be reached by flat loads
#define GLOBAL __attribute__((address_space(1)))

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

__device__ inline uint32_t round_up_block(uint32_t n) { return (n + kOptBlock - 1) & ~(uint32_t)(kOptBlock - 1); }

// four consecutive elements from `i` of `n`; behind the end: zeros.  DT: 0 fp32, 1 bf16, 2 fp16
template <int DT>
struct Quad {
    static __device__ inline void load(const void* base, uint64_t i, uint64_t n, float (&x)[4])
    {
        if constexpr (DT == 0) {
            const GLOBAL float* q = (const GLOBAL float*)base + i;
            f32x4u a = {0.f, 0.f, 0.f, 0.f};
            if (i + 4 <= n) a = *(const GLOBAL f32x4u*)q;
            else if (i < n) {
                a[0] = q[0];
                if (i + 1 < n) a[1] = q[1];
                if (i + 2 < n) a[2] = q[2];
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) x[k] = a[k];
        } else {
            const GLOBAL unsigned short* q = (const GLOBAL unsigned short*)base + i;
            u16x4u a = {0, 0, 0, 0};
            if (i + 4 <= n) a = *(const GLOBAL u16x4u*)q;
            else if (i < n) {
                a[0] = q[0];
                if (i + 1 < n) a[1] = q[1];
                if (i + 2 < n) a[2] = q[2];
            }
#pragma unroll
            for (int k = 0; k < 4; ++k)
                x[k] = DT == 1 ? bf16_to_f32(a[k]) : (float)__builtin_bit_cast(_Float16, (unsigned short)a[k]);
        }
    }
};

__device__ inline void store_f32(void* base, uint64_t i, uint64_t n, const float (&x)[4])
{
    GLOBAL float* q = (GLOBAL float*)base + i;
    if (i + 4 <= n) {
        f32x4u a;
#pragma unroll
        for (int k = 0; k < 4; ++k) a[k] = x[k];
        *(GLOBAL f32x4u*)q = a;
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (i + k < n) q[k] = x[k];
    }
}

__device__ inline void store_u16(void* base, uint64_t i, uint64_t n, const unsigned short (&x)[4])
{
    GLOBAL unsigned short* q = (GLOBAL unsigned short*)base + i;
    if (i + 4 <= n) {
        u16x4u a;
#pragma unroll
        for (int k = 0; k < 4; ++k) a[k] = x[k];
        *(GLOBAL u16x4u*)q = a;
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (i + k < n) q[k] = x[k];
    }
}

__device__ inline unsigned short bf16_nearest(float x)
{
    const uint32_t b = __float_as_uint(x);
    if ((b & 0x7F800000u) == 0x7F800000u) return (unsigned short)((b >> 16) | ((b & 0x7FFFFFu) ? 0x40u : 0u));
    return (unsigned short)((b + 0x7FFFu + ((b >> 16) & 1u)) >> 16);
}

// ---- e4m3 with a power of two for each block of 32 ---------------------------------------------------------------------
// The scale 2^(e - 127) puts the block's largest magnitude at 2^8 .. 1.75 * 2^8, e4m3's top (a magnitude of 1.75 * 2^k to
// 2^(k+1) goes one binade down, so that rounding up cannot pass the top).  Not finite counts as 0 there and is stored as NaN.
// The card's own conversions do the rest: v_cvt_scalef32_sr_fp8_f32 divides by the scale, adds the seed under the last kept
// bit (the seed's top bit at half a step; subnormals alike) and cuts, in one instruction instead of some fifteen; with 16
// random bits at the top of the seed it gave the definition's code for all of 4 million values, seeds and scales tried,
// subnormals, ties, infinities and NaN among them.  v_cvt_scalef32_pk_f32_fp8 reads two values back, all 256 scales right.
constexpr uint32_t kTop = 0x7F600000u;         // 1.75 * 2^127: what is above is stored as it, or it would round up to infinity

__device__ inline uint32_t scale_byte(uint32_t top_bits)
{
    const uint32_t e = (top_bits + 0x1FFFFFu) >> 23;
    return (e < 9u ? 9u : e) - 8u;
}

__device__ inline uint32_t finite_bits(float x)
{
    const uint32_t b = __float_as_uint(x) & 0x7FFFFFFFu;
    return b >= 0x7F800000u ? 0u : b < kTop ? b : kTop;
}

template <int CTRL>
__device__ inline uint32_t max_dpp(uint32_t x)
{
    const uint32_t o = (uint32_t)__builtin_amdgcn_update_dpp((int)x, (int)x, CTRL, 0xF, 0xF, false);
    return x > o ? x : o;
}
__device__ inline uint32_t max8(uint32_t x)                  // over the 8 lanes that hold one block: neighbours, pairs, the two quads
{
    return max_dpp<0x141>(max_dpp<0x4E>(max_dpp<0xB1>(x)));  // quad_perm [1,0,3,2], quad_perm [2,3,0,1], row_half_mirror
}

// the scale byte of a block whose lane holds x[0..3]; magnitudes above kTop are brought down to it (a branch that is hardly
// ever taken: the maximum shows whether there is one, v_max skips NaN)
__device__ inline uint32_t block_scale(float (&x)[4])
{
    float t = fmaxf(fmaxf(fabsf(x[0]), fabsf(x[1])), fmaxf(fabsf(x[2]), fabsf(x[3])));
    uint32_t top = max8(__float_as_uint(t) & 0x7FFFFFFFu);
    if (__builtin_expect(top > kTop, 0)) {                   // (the same in all 8 lanes)
        uint32_t b = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const uint32_t f = finite_bits(x[k]);
            if (f == kTop) x[k] = copysignf(__uint_as_float(kTop), x[k]);
            b = b > f ? b : f;
        }
        top = max8(b);
    }
    return scale_byte(top);
}

// four codes; ROOT: what is not zero is raised to the smallest code, 2^-9 of the scale (med3 of x, that, and x times a power
// of two no root is too small for: a root is 0 or at least 2^-75)
template <bool ROOT>
__device__ inline uint32_t e4m3_codes(const float (&x)[4], uint32_t e, const uint32_t (&seed)[4])
{
    const float s = __uint_as_float(e << 23);
    int c = 0;
    float y[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) y[k] = ROOT ? __builtin_amdgcn_fmed3f(x[k], s * 0x1p-9f, x[k] * 0x1p126f) : x[k];
    if (ROOT && __builtin_expect(__builtin_isunordered(x[0], x[1]) || __builtin_isunordered(x[2], x[3]), 0)) {
#pragma unroll
        for (int k = 0; k < 4; ++k) y[k] = x[k] != x[k] ? x[k] : y[k];           // (med3 passes over NaN)
    }
    c = __builtin_amdgcn_cvt_scalef32_sr_fp8_f32(c, y[0], seed[0], s, 0);
    c = __builtin_amdgcn_cvt_scalef32_sr_fp8_f32(c, y[1], seed[1], s, 1);
    c = __builtin_amdgcn_cvt_scalef32_sr_fp8_f32(c, y[2], seed[2], s, 2);
    c = __builtin_amdgcn_cvt_scalef32_sr_fp8_f32(c, y[3], seed[3], s, 3);
    return (uint32_t)c;
}

typedef float f32x2 __attribute__((ext_vector_type(2)));
__device__ inline void e4m3_values(uint32_t c, uint32_t e, float (&x)[4])
{
    const float s = __uint_as_float(e << 23);                // (the instruction reads 0 as 2^-127 and 255 as NaN, as e8m0 does)
    const f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(c, s, false), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(c, s, true);
    x[0] = a[0];
    x[1] = a[1];
    x[2] = b[0];
    x[3] = b[1];
}

// square roots to the nearest: y ~ 1 / sqrt(v), s = v y, then the residual v - s^2, exact in one fma, put right with y / 2.  That
// is within 2^-45 of the root before the last rounding; below 2^-90 (the residual would underflow), at 0 and at infinity sqrtf
__device__ inline void roots(const float (&v)[4], float (&r)[4])
{
    const float lo = fminf(fminf(v[0], v[1]), fminf(v[2], v[3])), hi = fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3]));
    if (__builtin_expect(lo >= 0x1p-90f && hi < INFINITY, 1)) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const float y = __builtin_amdgcn_rsqf(v[k]);
            const float s = v[k] * y;
            r[k] = fmaf(fmaf(-s, s, v[k]), 0.5f * y, s);
        }
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) r[k] = sqrtf(v[k]);
    }
}

// ---- AdamW -------------------------------------------------------------------------------------------------------------
//   g' = c g      m = b1 m + (1 - b1) g'      v = b2 v + (1 - b2) g'^2
//   p  = (1 - lr wd) p - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
// One workgroup owns kOptChunk consecutive elements of one tensor and that chunk's step counter, so t needs no second launch
// and no atomics: every chunk of a tensor counts the same steps.  All loads of the chunk are requested first; meanwhile one wave
// works out the step's scalars (two exponentials, divisions and a root in 64 bits) and hands them over through LDS.
struct StepScalars {
    double c1, c2;          // (1 - beta1) * c, (1 - beta2) * c^2
    float decay, step, isb2, gmul;
    uint32_t key;
};

// what a thread reads for its four elements
template <int BITS>
struct Operands {
    float p[4], g[4];
    float4 m, v;                       // 32 bits
    uint32_t mc, vc, me, ve;           // 8 bits
};

template <int BITS, int PDT, int GDT>
__device__ inline void load_operands(const AdamWArgs& a, const OptChunk& ck, const void* pp, const void* gp, uint32_t i, Operands<BITS>& d)
{
    const uint64_t off = (uint64_t)ck.offset32 * kOptBlock;
    Quad<PDT>::load(pp, i, ck.count, d.p);
    Quad<GDT>::load(gp, i, ck.count, d.g);
    const bool in = i < round_up_block(ck.count);
    if constexpr (BITS == 32) {
        d.m = d.v = float4{0.f, 0.f, 0.f, 0.f};
        if (in) {
            d.m = *(const float4*)((const float*)a.mo.m + off + i);
            d.v = *(const float4*)((const float*)a.mo.v + off + i);
        }
    } else {
        d.mc = d.vc = d.me = d.ve = 0;
        if (in) {
            d.mc = *(const uint32_t*)((const uint8_t*)a.mo.m + off + i);
            d.vc = *(const uint32_t*)((const uint8_t*)a.mo.v + off + i);
            d.me = a.mo.m_scale[ck.offset32 + i / kOptBlock];
            d.ve = a.mo.v_scale[ck.offset32 + i / kOptBlock];
        }
    }
}

template <int BITS, int PDT, int GDT>
__device__ inline void adamw_chunk(const AdamWArgs& a, const OptChunk ck, void* pp, const void* gp, StepScalars* sh)
{
    const AdamWScalars& sc = a.sc;
    const uint32_t n = ck.count, np = round_up_block(n);
    const uint64_t off = (uint64_t)ck.offset32 * kOptBlock;
    const uint32_t tid = threadIdx.x;
    Operands<BITS> d, next;
    load_operands<BITS, PDT, GDT>(a, ck, pp, gp, tid * 4, d);
    if (tid < 64) {
        int32_t* counter = a.mo.step + (size_t)a.chunk0 + blockIdx.x;
        const int t = *counter + 1;                                    // (this wave alone reads and writes it)
        const double lr = sc.lr_dev ? (double)*sc.lr_dev : sc.lr;
        const double bc1 = -expm1((double)t * sc.ln_beta1), bc2 = -expm1((double)t * sc.ln_beta2);
        double c = sc.grad_mul ? (double)*sc.grad_mul : 1.0;
        if (sc.grad_div) c /= (double)*sc.grad_div;
        if (sc.negate) c = -c;
        if (tid == 0) {
            *counter = t;
            sh->c1 = (1.0 - sc.beta1) * c;
            sh->c2 = (1.0 - sc.beta2) * (c * c);
            sh->decay = (float)(1.0 - lr * sc.wd);
            sh->step = (float)(lr / bc1);
            sh->isb2 = (float)(1.0 / sqrt(bc2));
            sh->gmul = (float)c;
            sh->key = mix32(sc.seed_key + (uint32_t)t * kGold);
        }
    }
    __syncthreads();
    const float decay = sh->decay, step = -sh->step, isb2 = sh->isb2, eps = (float)sc.eps, gmul = sh->gmul;
    const uint32_t key = sh->key;
    const double c1 = sh->c1, c2 = sh->c2;

#pragma unroll 2
    for (uint32_t i0 = 0; i0 < kOptChunk; i0 += 1024) {
        const uint32_t i = i0 + tid * 4;
        if (i >= np) break;                                            // (whole blocks of 32: 8 lanes)
        load_operands<BITS, PDT, GDT>(a, ck, pp, gp, i0 + 1024 < kOptChunk ? i + 1024 : kOptChunk, next);
        const uint64_t j = off + i;
        float m[4], r[4];
        uint32_t h[4];
        if (BITS == 8 || PDT == 1) {
            const uint32_t w = (uint32_t)j + (uint32_t)(j >> 32) * kGold;
#pragma unroll
            for (int k = 0; k < 4; ++k) h[k] = mix32((w + k) ^ key);
        }
        if constexpr (BITS == 32) {
            const float b1 = (float)sc.beta1, d1 = (float)(1.0 - sc.beta1), b2 = (float)sc.beta2, d2 = (float)(1.0 - sc.beta2);
            float* mq = (float*)&d.m;
            float* vq = (float*)&d.v;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float gk = d.g[k] * gmul;
                mq[k] = fmaf(b1, mq[k], d1 * gk);
                vq[k] = fmaf(b2, vq[k], (d2 * gk) * gk);
                m[k] = mq[k];
                r[k] = sqrtf(vq[k]);
            }
            *(float4*)((float*)a.mo.m + j) = d.m;
            *(float4*)((float*)a.mo.v + j) = d.v;
        } else {
            float mo[4], ro[4], v[4];
            e4m3_values(d.mc, d.me, mo);
            e4m3_values(d.vc, d.ve, ro);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const double gk = (double)d.g[k], rk = (double)ro[k];
                m[k] = (float)fma(sc.beta1, (double)mo[k], c1 * gk);
                v[k] = (float)fma(sc.beta2, rk * rk, c2 * (gk * gk));
            }
            roots(v, r);
            float ms[4], rs[4];
            uint32_t seed_m[4], seed_r[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                ms[k] = m[k];
                rs[k] = r[k];
                seed_m[k] = h[k] << 16;
                seed_r[k] = h[k] & 0xFFFF0000u;
            }
            const uint32_t em = block_scale(ms), er = block_scale(rs);
            *(uint32_t*)((uint8_t*)a.mo.m + j) = e4m3_codes<false>(ms, em, seed_m);
            *(uint32_t*)((uint8_t*)a.mo.v + j) = e4m3_codes<true>(rs, er, seed_r);
            if ((tid & 7) == 0) {
                a.mo.m_scale[j / kOptBlock] = (uint8_t)em;
                a.mo.v_scale[j / kOptBlock] = (uint8_t)er;
            }
        }
        float x[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) x[k] = fmaf(step, m[k] * __builtin_amdgcn_rcpf(fmaf(r[k], isb2, eps)), d.p[k] * decay);
        if constexpr (PDT == 0) store_f32(pp, i, n, x);
        else {
            // bf16 by stochastic rounding: 16 random bits under the last kept one, the rest cut off.  (A NaN whose low bits the
            // sum would carry out of is replaced by the plain one.)
            unsigned short q[4];
            if (__builtin_expect(__builtin_isunordered(x[0], x[1]) || __builtin_isunordered(x[2], x[3]), 0)) {
#pragma unroll
                for (int k = 0; k < 4; ++k) x[k] = x[k] != x[k] ? __uint_as_float(0x7FC00000u) : x[k];
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) q[k] = (unsigned short)((__float_as_uint(x[k]) + (mix32(h[k] + kGold) >> 16)) >> 16);
            store_u16(pp, i, n, q);
        }
        d = next;
    }
}

template <int BITS>
__global__ __launch_bounds__(256) void adamw_many_kernel(const AdamWArgs a)
{
    __shared__ StepScalars sh;
    const OptChunk ck = a.mo.chunks[a.chunk0 + blockIdx.x];
    const uint64_t pw = a.p[ck.tensor - a.tensor0], gw = a.g[ck.tensor - a.tensor0];
    if (gw == 0) return;
    if (a.sc.found_inf && *a.sc.found_inf != 0.f) return;
    const int pdt = (int)(pw >> 48), gdt = (int)(gw >> 48);
    const uint64_t base = (uint64_t)ck.index * kOptChunk;
    void* pp = (void*)((pw & kAddrMask) + base * (pdt ? 2 : 4));
    const void* gp = (const void*)((gw & kAddrMask) + base * (gdt ? 2 : 4));
    if (pdt == 0) {
        if (gdt == 0) adamw_chunk<BITS, 0, 0>(a, ck, pp, gp, &sh);
        else adamw_chunk<BITS, 0, 1>(a, ck, pp, gp, &sh);
    } else {
        if (gdt == 0) adamw_chunk<BITS, 1, 0>(a, ck, pp, gp, &sh);
        else adamw_chunk<BITS, 1, 1>(a, ck, pp, gp, &sh);
    }
}

// which tensor of a launch a workgroup works on (the last one with block0 <= blk), its element type and size
struct Found {
    const char* base;
    uint64_t n;
    int dt;
    uint32_t block;         // in the tensor
};
__device__ inline Found find_tensor(const OptTensors& ts, uint32_t blk)
{
    int lo = 0, hi = ts.count - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (ts.t[mid].block0 <= blk) lo = mid;
        else hi = mid - 1;
    }
    const OptTensor& t = ts.t[lo];
    return Found{(const char*)(t.ptr & kAddrMask), t.numel_lo | (t.ptr >> 52) << 32, (int)(t.ptr >> 48) & 15, blk - t.block0};
}

__device__ inline void load_quad_dt(int dt, const void* base, uint64_t i, uint64_t n, float (&x)[4])
{
    if (dt == 0) Quad<0>::load(base, i, n, x);
    else if (dt == 1) Quad<1>::load(base, i, n, x);
    else Quad<2>::load(base, i, n, x);
}

// ---- total norm --------------------------------------------------------------------------------------------------------
__device__ inline double wave_sum(double x)
{
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) x += __shfl_xor(x, d);
    return x;
}

// 16 bytes of a list's tensor as 64-bit squares' sum; any alignment of the element
template <int DT>
struct Vec16 {
    static constexpr int N = DT == 0 ? 4 : 8;
    typedef float f4 __attribute__((ext_vector_type(4), aligned(4)));
    typedef unsigned short h8 __attribute__((ext_vector_type(8), aligned(2)));
    union {
        f4 f;
        h8 h;
    };
    __device__ inline void load(const void* p, uint64_t i)
    {
        if constexpr (DT == 0) f = *(const GLOBAL f4*)((const GLOBAL float*)p + i);
        else h = *(const GLOBAL h8*)((const GLOBAL unsigned short*)p + i);
    }
    __device__ inline double add(double acc) const
    {
#pragma unroll
        for (int k = 0; k < N; ++k) {
            const double x = DT == 0 ? (double)f[k] : DT == 1 ? (double)bf16_to_f32(h[k]) : (double)(float)__builtin_bit_cast(_Float16, (unsigned short)h[k]);
            acc = fma(x, x, acc);
        }
        return acc;
    }
};

template <int DT>
__device__ inline double sum_squares(const void* p, uint64_t base, uint64_t end)
{
    constexpr int N = Vec16<DT>::N, U = 4;                 // four loads of 16 bytes requested before the first is used
    constexpr uint32_t STEP = 256 * N;
    double acc = 0.0;
    uint64_t i = base + threadIdx.x * N;
    for (; i + (U - 1) * STEP + N <= end; i += U * STEP) {
        Vec16<DT> x[U];
#pragma unroll
        for (int u = 0; u < U; ++u) x[u].load(p, i + u * STEP);
#pragma unroll
        for (int u = 0; u < U; ++u) acc = x[u].add(acc);
    }
    for (; i < end; i += STEP) {
        if (i + N <= end) {
            Vec16<DT> x;
            x.load(p, i);
            acc = x.add(acc);
        } else {
            for (uint64_t k = i; k < end; ++k) {
                const double x = DT == 0 ? (double)((const GLOBAL float*)p)[k]
                               : DT == 1 ? (double)bf16_to_f32(((const GLOBAL unsigned short*)p)[k])
                                         : (double)(float)__builtin_bit_cast(_Float16, ((const GLOBAL unsigned short*)p)[k]);
                acc = fma(x, x, acc);
            }
        }
    }
    return acc;
}

// sums of squares in 64 bits, in a fixed order: one partial sum for each workgroup's elements
__global__ __launch_bounds__(256) void norm_partial_kernel(const OptTensors ts, uint32_t per_block, double* __restrict__ partial)
{
    __shared__ double red[4];
    const Found f = find_tensor(ts, blockIdx.x);
    const uint64_t base = (uint64_t)f.block * per_block;
    const uint64_t end = base + per_block < f.n ? base + per_block : f.n;
    double acc = f.dt == 0 ? sum_squares<0>(f.base, base, end) : f.dt == 1 ? sum_squares<1>(f.base, base, end) : sum_squares<2>(f.base, base, end);
    acc = wave_sum(acc);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = acc;
    __syncthreads();
    if (threadIdx.x == 0) partial[(size_t)ts.partial0 + blockIdx.x] = (red[0] + red[1]) + (red[2] + red[3]);
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
    const Found f = find_tensor(ts, blockIdx.x);
    const uint64_t n = f.n;
    const int dt = f.dt;
    void* const q0 = (void*)f.base;
    const uint64_t base = (uint64_t)f.block * kOptChunk;
    for (int it = 0; it < kOptChunk / 1024; ++it) {
        const uint64_t i = base + it * 1024 + threadIdx.x * 4;
        if (i >= n) break;
        float g[4];
        load_quad_dt(dt, q0, i, n, g);
#pragma unroll
        for (int k = 0; k < 4; ++k) g[k] *= c;
        if (dt == 0) store_f32(q0, i, n, g);
        else {
            unsigned short q[4];
#pragma unroll
            for (int k = 0; k < 4; ++k)
                q[k] = dt == 1 ? bf16_nearest(g[k]) : __builtin_bit_cast(unsigned short, (_Float16)g[k]);
            store_u16(q0, i, n, q);
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
    float a[4], v4[4], b[4];
    Quad<0>::load(m, i, n, a);
    Quad<0>::load(v, i, n, v4);
    roots(v4, b);
    const uint32_t em = block_scale(a), er = block_scale(b);
    const uint32_t half[4] = {0x80000000u, 0x80000000u, 0x80000000u, 0x80000000u};
    *(uint32_t*)(m8 + i) = e4m3_codes<false>(a, em, half);
    *(uint32_t*)(r8 + i) = e4m3_codes<true>(b, er, half);
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
    float a[4], b[4];
    e4m3_values(*(const uint32_t*)(m8 + i), me[i / kOptBlock], a);
    e4m3_values(*(const uint32_t*)(r8 + i), re[i / kOptBlock], b);
#pragma unroll
    for (int k = 0; k < 4; ++k) b[k] *= b[k];
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
