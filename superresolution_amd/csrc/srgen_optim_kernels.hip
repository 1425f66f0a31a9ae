// srgen_optim_kernels.hip -- optimizer operators over a list of tensors: AdamW with moments in 32 or 8 bits, the total
// gradient norm, scaling in place, and moments written to / read from 8 bits.
#include "srgen_optim.h"

namespace srgen {
namespace {

// an address that came as a number is in device memory: without this it would be reached by flat loads
#define GLOBAL __attribute__((address_space(1)))

// unaligned vectors: a gradient that is a view into a flat buffer starts at any element (global loads need element alignment only)
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
template <int V>
struct HalfVec;
template <>
struct HalfVec<4> {
    typedef unsigned short type __attribute__((ext_vector_type(4)));
    typedef unsigned short unaligned __attribute__((ext_vector_type(4), aligned(2)));
    typedef uint32_t codes __attribute__((ext_vector_type(1), aligned(4)));
};
template <>
struct HalfVec<8> {
    typedef unsigned short type __attribute__((ext_vector_type(8)));
    typedef unsigned short unaligned __attribute__((ext_vector_type(8), aligned(2)));
    typedef uint32_t codes __attribute__((ext_vector_type(2), aligned(4)));
};
template <int V>
using Codes = typename HalfVec<V>::codes;      // V e4m3 values, four to a word

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

template <bool NT, typename T>
__device__ inline T load_as(const GLOBAL T* p)
{
    if constexpr (NT) return __builtin_nontemporal_load(p);
    else return *p;
}
template <bool NT, typename T>
__device__ inline void store_as(T x, GLOBAL T* p)
{
    if constexpr (NT) __builtin_nontemporal_store(x, p);
    else *p = x;
}

// V consecutive elements as they are in memory (values() converts: a conversion beside the load would wait for it).
// DT: 0 fp32, 1 bf16, 2 fp16.
template <int DT, int V>
struct Elements {
    typename HalfVec<V>::type h;
    __device__ inline void values(float (&x)[V]) const
    {
#pragma unroll
        for (int k = 0; k < V; ++k)
            x[k] = DT == 1 ? bf16_to_f32(h[k]) : (float)__builtin_bit_cast(_Float16, (unsigned short)h[k]);
    }
};
template <int V>
struct Elements<0, V> {
    f32x4 f[V / 4];
    __device__ inline void values(float (&x)[V]) const
    {
#pragma unroll
        for (int k = 0; k < V; ++k) x[k] = f[k / 4][k % 4];
    }
};

// elements i .. i + V - 1 of `n`; behind the end: zeros.  FULL: all are there.  The index counts from a base that is the same for
// the workgroup, in 32 bits.
template <int DT, int V, bool FULL, bool NT>
__device__ inline Elements<DT, V> load_elements(const void* base, uint32_t i, uint32_t n)
{
    Elements<DT, V> a;
    if constexpr (DT == 0) {
        const GLOBAL float* q = (const GLOBAL float*)base + i;
#pragma unroll
        for (int u = 0; u < V / 4; ++u) {
            if (!FULL) a.f[u] = f32x4{0.f, 0.f, 0.f, 0.f};
            const uint32_t at = i + 4 * u;
            if (FULL || at + 4 <= n) a.f[u] = load_as<NT>((const GLOBAL f32x4u*)(q + 4 * u));
            else if (at < n) {
                a.f[u][0] = q[4 * u];
                if (at + 1 < n) a.f[u][1] = q[4 * u + 1];
                if (at + 2 < n) a.f[u][2] = q[4 * u + 2];
            }
        }
    } else {
        const GLOBAL unsigned short* q = (const GLOBAL unsigned short*)base + i;
        if (FULL || i + V <= n) a.h = load_as<NT>((const GLOBAL typename HalfVec<V>::unaligned*)q);
        else {
#pragma unroll
            for (int k = 0; k < V; ++k) a.h[k] = i + k < n ? q[k] : (unsigned short)0;
        }
    }
    return a;
}

template <int V, bool FULL, bool NT>
__device__ inline void store_f32(void* base, uint32_t i, uint32_t n, const float (&x)[V])
{
    GLOBAL float* q = (GLOBAL float*)base + i;
    if (FULL || i + V <= n) {
#pragma unroll
        for (int u = 0; u < V / 4; ++u) store_as<NT>(f32x4u{x[4 * u], x[4 * u + 1], x[4 * u + 2], x[4 * u + 3]}, (GLOBAL f32x4u*)(q + 4 * u));
    } else {
#pragma unroll
        for (int k = 0; k < V; ++k)
            if (i + k < n) q[k] = x[k];
    }
}

template <int V, bool FULL, bool NT>
__device__ inline void store_u16(void* base, uint32_t i, uint32_t n, const unsigned short (&x)[V])
{
    GLOBAL unsigned short* q = (GLOBAL unsigned short*)base + i;
    if (FULL || i + V <= n) {
        typename HalfVec<V>::unaligned a;
#pragma unroll
        for (int k = 0; k < V; ++k) a[k] = x[k];
        store_as<NT>(a, (GLOBAL typename HalfVec<V>::unaligned*)q);
    } else {
#pragma unroll
        for (int k = 0; k < V; ++k)
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
constexpr uint32_t kLow = (9u << 23) - 0x1FFFFFu;  // a maximum below this counts as this: the scale is then 2^-126, the lowest

__device__ inline uint32_t finite_bits(float x)
{
    const uint32_t b = __float_as_uint(x) & 0x7FFFFFFFu;
    return b >= 0x7F800000u ? 0u : b < kTop ? b : kTop;
}

template <int CTRL>
__device__ inline uint32_t max_dpp(uint32_t x)
{
    const uint32_t o = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, 0xF, 0xF, false);   // (0: one instruction with the max)
    return x > o ? x : o;
}
// over the 32 / V lanes that hold one block: neighbours, pairs and, of 8, the two quads
template <int V>
__device__ inline uint32_t max_block(uint32_t x)
{
    x = max_dpp<0x4E>(max_dpp<0xB1>(x));                     // quad_perm [1,0,3,2], quad_perm [2,3,0,1]
    return V == 4 ? max_dpp<0x141>(x) : x;                   // row_half_mirror
}

__device__ inline uint32_t max_u32(uint32_t a, uint32_t b) { return a > b ? a : b; }

// The scale (as a float's bits) of a block whose lane holds x[0 .. V-1]; magnitudes above kTop are brought down to it, in a branch
// that is hardly ever taken (v_max skips NaN; in a root's bits NaN is above everything).  ROOT: no x is negative.
template <int V, bool ROOT>
__device__ inline uint32_t block_scale(float (&x)[V])
{
    uint32_t t;
    if constexpr (ROOT) {
        t = kLow;
#pragma unroll
        for (int k = 0; k < V; k += 2) t = max_u32(max_u32(t, __float_as_uint(x[k])), __float_as_uint(x[k + 1]));
    } else {
        float f = __uint_as_float(kLow);
#pragma unroll
        for (int k = 0; k < V; k += 2) f = fmaxf(fmaxf(f, fabsf(x[k])), fabsf(x[k + 1]));
        t = __float_as_uint(f);
    }
    uint32_t top = max_block<V>(t);
    if (__builtin_expect(top > kTop, 0)) {                   // (the same in all lanes of the block)
        uint32_t b = kLow;
#pragma unroll
        for (int k = 0; k < V; ++k) {
            const uint32_t f = finite_bits(x[k]);
            if (f == kTop) x[k] = copysignf(__uint_as_float(kTop), x[k]);
            b = max_u32(b, f);
        }
        top = max_block<V>(b);
    }
    return ((top + 0x1FFFFFu) & 0x7F800000u) - (8u << 23);
}

template <int V>
__device__ inline Codes<V> e4m3_codes(const float (&x)[V], uint32_t scale, const uint32_t (&seed)[V])
{
    const float s = __uint_as_float(scale);
    Codes<V> out;
#pragma unroll
    for (int u = 0; u < V; u += 4) {
        int c = 0;
        c = __builtin_amdgcn_cvt_scalef32_sr_fp8_f32(c, x[u], seed[u], s, 0);
        c = __builtin_amdgcn_cvt_scalef32_sr_fp8_f32(c, x[u + 1], seed[u + 1], s, 1);
        c = __builtin_amdgcn_cvt_scalef32_sr_fp8_f32(c, x[u + 2], seed[u + 2], s, 2);
        c = __builtin_amdgcn_cvt_scalef32_sr_fp8_f32(c, x[u + 3], seed[u + 3], s, 3);
        out[u / 4] = (uint32_t)c;
    }
    return out;
}

// the same for roots: what is not zero is raised to the smallest code, 2^-9 of the scale.  `plain`: none is 0 or NaN (roots())
template <int V>
__device__ inline Codes<V> e4m3_root_codes(const float (&x)[V], bool plain, uint32_t scale, const uint32_t (&seed)[V])
{
    const float q = __uint_as_float(scale) * 0x1p-9f;
    float y[V];
    if (__builtin_expect(plain, 1)) {
#pragma unroll
        for (int k = 0; k < V; ++k) y[k] = __uint_as_float(max_u32(__float_as_uint(x[k]), __float_as_uint(q)));  // (whole numbers: no care for NaN)
    } else {
#pragma unroll
        for (int k = 0; k < V; ++k) y[k] = x[k] > 0.f && x[k] < q ? q : x[k];
    }
    return e4m3_codes<V>(y, scale, seed);
}

typedef float f32x2 __attribute__((ext_vector_type(2)));
template <int V>
__device__ inline void e4m3_values(Codes<V> c, uint32_t e, float (&x)[V])
{
    const float s = __uint_as_float(e << 23);                // (the instruction reads 0 as 2^-127 and 255 as NaN, as e8m0 does)
#pragma unroll
    for (int u = 0; u < V; u += 4) {
        const f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(c[u / 4], s, false), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(c[u / 4], s, true);
        x[u] = a[0];
        x[u + 1] = a[1];
        x[u + 2] = b[0];
        x[u + 3] = b[1];
    }
}

// Square roots to the nearest: y ~ 1 / sqrt(v), s = v y, then the residual v - s^2, exact in one fma, put right with y / 2.
// That is within 2^-45 of the root before the last rounding.  Below 2^-90 (the residual would underflow), at 0, infinity and NaN
// sqrtf instead; returns whether there was none of these.
template <int V>
__device__ inline bool roots(const float (&v)[V], float (&r)[V])
{
    float lo = v[0], hi = v[0];
    bool plain = true;
#pragma unroll
    for (int k = 0; k < V; k += 2) {
        lo = fminf(fminf(lo, v[k]), v[k + 1]);
        hi = fmaxf(fmaxf(hi, v[k]), v[k + 1]);
        plain = plain && !__builtin_isunordered(v[k], v[k + 1]);
    }
    plain = plain && lo >= 0x1p-90f && hi < INFINITY;
    if (__builtin_expect(plain, 1)) {
#pragma unroll
        for (int k = 0; k < V; ++k) {
            const float y = __builtin_amdgcn_rsqf(v[k]);
            const float s = v[k] * y;
            r[k] = fmaf(fmaf(-s, s, v[k]), 0.5f * y, s);
        }
    } else {
#pragma unroll
        for (int k = 0; k < V; ++k) r[k] = sqrtf(v[k]);
    }
    return plain;
}

// ---- norm and clip coefficient from partial sums -----------------------------------------------------------------------
__device__ inline double wave_sum(double x)
{
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) x += __shfl_xor(x, d);
    return x;
}

// the sum of up to kOptWavePartials numbers by one wave, in a fixed order; all its loads are requested at once
__device__ inline double wave_total(const double* __restrict__ partial, uint32_t n)
{
    constexpr int U = kOptWavePartials / 64;
    const uint32_t lane = threadIdx.x & 63;
    double x[U], acc = 0.0;
#pragma unroll
    for (int u = 0; u < U; ++u) x[u] = lane + 64 * u < n ? partial[lane + 64 * u] : 0.0;
#pragma unroll
    for (int u = 0; u < U; ++u) acc += x[u];
    return wave_sum(acc);
}

// {sqrt(sum), min(1, max_norm / (norm + 1e-6))}; a NaN norm gives a NaN coefficient
struct NormCoef {
    float norm, coef;
};
__device__ inline NormCoef norm_coef_of(double sum, double max_norm)
{
    const float norm = (float)sqrt(sum);
    const double c = max_norm / ((double)norm + 1e-6);
    return NormCoef{norm, c > 1.0 ? 1.f : (float)c};
}

// ---- AdamW -------------------------------------------------------------------------------------------------------------
//   g' = c g      m = b1 m + (1 - b1) g'      v = b2 v + (1 - b2) g'^2
//   p  = (1 - lr wd) p - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
// One workgroup owns kOptChunk consecutive elements of one tensor and that chunk's step counter, so t needs no second launch
// and no atomics: every chunk of a tensor counts the same steps.  The first loads are requested before anything else; meanwhile
// one wave works out the step's scalars (two exponentials, divisions and a root in 64 bits) and hands them over through LDS.
// A thread takes V elements at a time: 4, or 8 of bf16 with 8-bit moments, where the arithmetic is what takes the time and half
// as many threads to a block of 32 make its scale cheaper (268M parameters: 540 -> 494 us).
// What bounds it: memory (32 bits: 28 bytes an fp32 element, 268M in 1,305 us = 5.76 TB/s, vector units 19 % busy; 8 bits fp32: 16
// bytes, 5.5 TB/s at 50 %), but for 8 bits with bf16 parameters (10 bytes and 56 vector instructions an element, 268M in 479 to 494 us,
// by the card, = 5.5 to 5.7 TB/s at 97 % busy).  In cache (3.2M fp32, 32 bits) 16 us = 5.6 TB/s; a single workgroup 4.2 us, most of it the launch.
struct StepScalars {
    double c1, c2;          // (1 - beta1) * c, (1 - beta2) * c^2
    float decay;            // 1 - lr wd
    float ra, rb;           // p - m / (ra r + rb): 1 / (s sqrt(1 - b2^t)) and eps / s with the step size s = lr / (1 - b1^t)
    float gmul;
    uint32_t key;
};

// (the same for the workgroup: in scalar registers)
__device__ inline uint32_t uniform(uint32_t x) { return (uint32_t)__builtin_amdgcn_readfirstlane((int)x); }
__device__ inline float uniform(float x) { return __uint_as_float(uniform(__float_as_uint(x))); }
__device__ inline double uniform(double x)
{
    const uint64_t b = __builtin_bit_cast(uint64_t, x);
    return __builtin_bit_cast(double, (uint64_t)uniform((uint32_t)b) | (uint64_t)uniform((uint32_t)(b >> 32)) << 32);
}
__device__ inline StepScalars uniform(const StepScalars& s)
{
    return StepScalars{uniform(s.c1), uniform(s.c2), uniform(s.decay), uniform(s.ra), uniform(s.rb), uniform(s.gmul), uniform(s.key)};
}

// what a thread reads for its V elements
template <int BITS, int PDT, int GDT, int V>
struct Operands {
    Elements<PDT, V> p;
    Elements<GDT, V> g;
    Elements<0, V> m, v;               // 32 bits
    Codes<V> mc, vc;                   // 8 bits
    uint32_t me, ve;
};

// a chunk's operands: bases are the same for the workgroup, indexes count from them
struct Chunk {
    void* p;
    const void* g;
    uint8_t* m;                        // (bytes)
    uint8_t* v;
    uint8_t* me;
    uint8_t* ve;
    uint32_t n, np;                    // elements; the same in whole blocks of 32
    uint32_t lo, w;                    // position: its low word; that with the high word mixed in
    bool first;                        // of its tensor
};

template <int BITS, int PDT, int GDT, int V, bool FULL, bool NT>
__device__ inline void load_operands(const Chunk& c, uint32_t i, Operands<BITS, PDT, GDT, V>& d)
{
    d.p = load_elements<PDT, V, FULL, NT>(c.p, i, c.n);
    d.g = load_elements<GDT, V, FULL, NT>(c.g, i, c.n);
    if constexpr (BITS == 32) {
        d.m = load_elements<0, V, FULL, NT>(c.m, i, c.np);
        d.v = load_elements<0, V, FULL, NT>(c.v, i, c.np);
    } else {
        if (!FULL) {
            d.mc = d.vc = 0;
            d.me = d.ve = 0;
        }
        if (FULL || i < c.np) {
            d.mc = load_as<NT>((const GLOBAL Codes<V>*)(c.m + i));
            d.vc = load_as<NT>((const GLOBAL Codes<V>*)(c.v + i));
            d.me = ((const GLOBAL uint8_t*)c.me)[i / kOptBlock];
            d.ve = ((const GLOBAL uint8_t*)c.ve)[i / kOptBlock];
        }
    }
}

template <int BITS, int PDT, int GDT, int V, bool FULL, bool NT>
__device__ inline void update(const AdamWScalars& sc, const StepScalars& sh, const Chunk& c, uint32_t i, const Operands<BITS, PDT, GDT, V>& d)
{
    float m[V], r[V], p[V], g[V];
    uint32_t h[V];
    bool plain = true;
    d.g.values(g);
    d.p.values(p);
    if (BITS == 8 || PDT == 1) {
        uint32_t w = c.w + i;
        if (!FULL && c.lo + i < c.lo) w += kGold;                      // (the high word goes up inside the chunk)
#pragma unroll
        for (int k = 0; k < V; ++k) h[k] = mix32((w + k) ^ sh.key);
    }
    if constexpr (BITS == 32) {
        const float b1 = (float)sc.beta1, d1 = (float)(1.0 - sc.beta1), b2 = (float)sc.beta2, d2 = (float)(1.0 - sc.beta2);
        float v[V];
        d.m.values(m);
        d.v.values(v);
#pragma unroll
        for (int k = 0; k < V; ++k) {
            const float gk = g[k] * sh.gmul;
            m[k] = fmaf(b1, m[k], d1 * gk);
            v[k] = fmaf(b2, v[k], (d2 * gk) * gk);
            r[k] = sqrtf(v[k]);
        }
        store_f32<V, true, NT>(c.m, i, 0, m);                          // (the padding of the last block is there)
        store_f32<V, true, NT>(c.v, i, 0, v);
    } else {
        float mo[V], ro[V], v[V];
        e4m3_values<V>(d.mc, d.me, mo);
        e4m3_values<V>(d.vc, d.ve, ro);
#pragma unroll
        for (int k = 0; k < V; ++k) {
            const double gk = (double)g[k], rk = (double)ro[k];
            m[k] = (float)fma(sc.beta1, (double)mo[k], sh.c1 * gk);
            v[k] = (float)fma(sc.beta2, rk * rk, sh.c2 * (gk * gk));
        }
        plain = roots<V>(v, r);
    }
    float x[V];
#pragma unroll
    for (int k = 0; k < V; ++k) x[k] = fmaf(-m[k], __builtin_amdgcn_rcpf(fmaf(r[k], sh.ra, sh.rb)), p[k] * sh.decay);
    if constexpr (PDT == 0) store_f32<V, FULL, NT>(c.p, i, c.n, x);
    else {
        // bf16 by stochastic rounding: 16 random bits under the last kept one, the rest cut off.  (A NaN whose low bits the sum
        // would carry out of is replaced by the plain one.)
        unsigned short q[V];
        bool nan = false;
#pragma unroll
        for (int k = 0; k < V; k += 2) nan = nan || __builtin_isunordered(x[k], x[k + 1]);
        if (__builtin_expect(nan, 0)) {
#pragma unroll
            for (int k = 0; k < V; ++k) x[k] = x[k] != x[k] ? __uint_as_float(0x7FC00000u) : x[k];
        }
#pragma unroll
        for (int k = 0; k < V; ++k) q[k] = (unsigned short)((__float_as_uint(x[k]) + (mix32(h[k] + kGold) >> 16)) >> 16);
        store_u16<V, FULL, NT>(c.p, i, c.n, q);
    }
    if constexpr (BITS == 8) {
        uint32_t seed_m[V], seed_r[V];
#pragma unroll
        for (int k = 0; k < V; ++k) {
            seed_m[k] = h[k] << 16;
            seed_r[k] = h[k] & 0xFFFF0000u;
        }
        const uint32_t em = block_scale<V, false>(m), er = block_scale<V, true>(r);
        store_as<NT>(e4m3_codes<V>(m, em, seed_m), (GLOBAL Codes<V>*)(c.m + i));
        store_as<NT>(e4m3_root_codes<V>(r, plain, er, seed_r), (GLOBAL Codes<V>*)(c.v + i));
        if ((i & (kOptBlock - 1)) == 0) {
            ((GLOBAL uint8_t*)c.me)[i / kOptBlock] = (uint8_t)(em >> 23);
            ((GLOBAL uint8_t*)c.ve)[i / kOptBlock] = (uint8_t)(er >> 23);
        }
    }
}

template <int BITS, int PDT, int GDT, int V, bool FULL, bool NT>
__device__ inline void adamw_chunk(const AdamWArgs& a, const Chunk& c, StepScalars* shared)
{
    constexpr uint32_t STRIDE = 256 * V;
    const AdamWScalars& sc = a.sc;
    const uint32_t tid = threadIdx.x;
    Operands<BITS, PDT, GDT, V> d, next;
    load_operands<BITS, PDT, GDT, V, FULL, NT>(c, tid * V, d);
    if (tid < 64) {
        int32_t* counter = a.mo.step + (size_t)a.chunk0 + blockIdx.x;
        const int t = *counter + 1;                                    // (this wave alone reads and writes it)
        const double lr = sc.lr_dev ? (double)*sc.lr_dev : sc.lr;
        const double bc1 = -expm1((double)t * sc.ln_beta1), bc2 = -expm1((double)t * sc.ln_beta2);
        const double s = lr / bc1;
        double f = sc.grad_mul ? (double)*sc.grad_mul : 1.0;
        if (sc.partial) {
            const NormCoef r = norm_coef_of(wave_total(sc.partial, sc.partials), sc.max_norm);
            f = (double)r.coef;
            if (tid == 0 && c.first) {                                 // (of every tensor that takes the step: the same values)
                sc.norm_coef[0] = r.norm;
                sc.norm_coef[1] = r.coef;
            }
        }
        if (sc.grad_div) f /= (double)*sc.grad_div;
        if (sc.negate) f = -f;
        if (tid == 0) {
            *counter = t;
            shared->c1 = (1.0 - sc.beta1) * f;
            shared->c2 = (1.0 - sc.beta2) * (f * f);
            shared->decay = (float)(1.0 - lr * sc.wd);
            // (a step size of 0 or next to it: an infinite denominator, by a finite factor that is not 0, so that neither a root of 0
            // nor an infinite one makes NaN of it; the reciprocal takes a subnormal for 0)
            shared->ra = (float)fmin(1.0 / (s * sqrt(bc2)), 3.0e38);
            shared->rb = s == 0.0 ? INFINITY : sc.eps == 0.0 ? 0.f : (float)fmax(sc.eps / s, 0x1p-126);
            shared->gmul = (float)f;
            shared->key = mix32(sc.seed_key + (uint32_t)t * kGold);
        }
    }
    __syncthreads();
    const StepScalars sh = uniform(*shared);
    if constexpr (FULL) {
#pragma unroll 2
        for (uint32_t i0 = 0; i0 < kOptChunk; i0 += STRIDE) {
            if (i0 + STRIDE < kOptChunk) load_operands<BITS, PDT, GDT, V, FULL, NT>(c, i0 + STRIDE + tid * V, next);
            update<BITS, PDT, GDT, V, FULL, NT>(sc, sh, c, i0 + tid * V, d);
            d = next;
        }
    } else {
#pragma unroll 1
        for (uint32_t i = tid * V; i < c.np; i += STRIDE) {
            if (i >= STRIDE) load_operands<BITS, PDT, GDT, V, FULL, NT>(c, i, d);
            update<BITS, PDT, GDT, V, FULL, NT>(sc, sh, c, i, d);
        }
    }
}

template <int BITS, int PDT, int GDT, int V, bool NT>
__device__ inline void adamw_chunk_any(const AdamWArgs& a, const Chunk& c, StepScalars* shared)
{
    if (c.n == kOptChunk && c.lo + (kOptChunk - 1) >= c.lo) adamw_chunk<BITS, PDT, GDT, V, true, NT>(a, c, shared);
    else adamw_chunk<BITS, PDT, GDT, V, false, NT>(a, c, shared);
}

// LIST: types of the list's parameters and gradients: 0 all fp32, 1 all bf16, 2 mixed.  Kernels of their own for the first two leave
// each the registers that its own path needs: 6 workgroups a CU instead of 4 for fp32 with 8 bits (discriminator's step 18.2 -> 17.5
// us), 5 instead of 4 for bf16 (268M parameters 498 -> 484 us).
template <int BITS, int LIST, bool NT>
__global__ __launch_bounds__(256) void adamw_many_kernel(const AdamWArgs a)
{
    __shared__ StepScalars shared;
    const OptChunk ck = a.mo.chunks[a.chunk0 + blockIdx.x];
    const uint32_t at = ck.tensor - a.tensor0, hi = a.hi[at];
    const uint64_t pw = a.p[at] | (uint64_t)(hi & 0xFFFFu) << 32, gw = a.g[at] | (uint64_t)(hi >> 16) << 32;
    if (gw == 0) return;
    if (a.sc.found_inf && *a.sc.found_inf != 0.f) return;
    const int pdt = LIST == 2 ? (int)(pw & 1) : LIST, gdt = LIST == 2 ? (int)(gw & 1) : LIST;
    const uint64_t base = (uint64_t)ck.index * kOptChunk, off = (uint64_t)ck.offset32 * kOptBlock;
    const Chunk c{(void*)((pw & ~1ull) + base * (pdt ? 2 : 4)), (const void*)((gw & ~1ull) + base * (gdt ? 2 : 4)),
                  (uint8_t*)a.mo.m + off * (BITS / 8), (uint8_t*)a.mo.v + off * (BITS / 8), a.mo.m_scale + ck.offset32, a.mo.v_scale + ck.offset32,
                  ck.count, round_up_block(ck.count), (uint32_t)off, (uint32_t)off + (uint32_t)(off >> 32) * kGold, ck.index == 0};
    if constexpr (LIST == 0) adamw_chunk_any<BITS, 0, 0, 4, NT>(a, c, &shared);
    else if constexpr (LIST == 1) adamw_chunk_any<BITS, 1, 1, BITS == 8 ? 8 : 4, NT>(a, c, &shared);
    else if (pdt == 0) {
        if (gdt == 0) adamw_chunk_any<BITS, 0, 0, 4, NT>(a, c, &shared);
        else adamw_chunk_any<BITS, 0, 1, 4, NT>(a, c, &shared);
    } else {
        if (gdt == 0) adamw_chunk_any<BITS, 1, 0, 4, NT>(a, c, &shared);
        else adamw_chunk_any<BITS, 1, 1, 4, NT>(a, c, &shared);
    }
}

// which part of which tensor a workgroup works on
struct Found {
    const char* base;       // of the part
    uint32_t n;             // its elements
    int dt;
};
// (every wave counts the tensors that start at or before the workgroup: its loads go out at once, a search's would follow each other)
__device__ inline Found find_part(const OptTensors& ts, uint32_t blk)
{
    const int lane = threadIdx.x & 63;
    int at = -1;
#pragma unroll
    for (int u = 0; u < (kOptMaxListed + 63) / 64; ++u) {
        const int k = lane + 64 * u;
        const uint32_t first = ts.block0[k < kOptMaxListed ? k : 0];
        at += __popcll(__ballot(k < ts.count && first <= blk));
    }
    at = __builtin_amdgcn_readfirstlane(at);
    const uint64_t t = ts.t[at];
    const int dt = (int)(t >> 48) & 3;
    return Found{(const char*)(t & kAddrMask) + (uint64_t)(blk - ts.block0[at]) * ts.part * (dt == 0 ? 4 : 2),
                 blk + 1 == ts.block0[at + 1] ? (uint32_t)(t >> 50) + 1 : ts.part, dt};
}

// ---- total norm --------------------------------------------------------------------------------------------------------
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
    template <bool NT>
    __device__ inline void load(const void* p, uint32_t i)
    {
        if constexpr (DT == 0) f = load_as<NT>((const GLOBAL f4*)((const GLOBAL float*)p + i));
        else h = load_as<NT>((const GLOBAL h8*)((const GLOBAL unsigned short*)p + i));
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

template <int DT, bool NT>
__device__ inline double sum_squares(const void* p, uint32_t n)
{
    constexpr int N = Vec16<DT>::N, U = 4;                 // four loads of 16 bytes requested before the first is used
    constexpr uint32_t STEP = 256 * N;
    double acc = 0.0;
    uint32_t i = threadIdx.x * N;
    for (; i + (U - 1) * STEP + N <= n; i += U * STEP) {
        Vec16<DT> x[U];
#pragma unroll
        for (int u = 0; u < U; ++u) x[u].template load<NT>(p, i + u * STEP);
#pragma unroll
        for (int u = 0; u < U; ++u) acc = x[u].add(acc);
    }
    for (; i < n; i += STEP) {
        if (i + N <= n) {
            Vec16<DT> x;
            x.template load<NT>(p, i);
            acc = x.add(acc);
        } else {
            for (uint32_t k = i; k < n; ++k) {
                const double x = DT == 0 ? (double)((const GLOBAL float*)p)[k]
                               : DT == 1 ? (double)bf16_to_f32(((const GLOBAL unsigned short*)p)[k])
                                         : (double)(float)__builtin_bit_cast(_Float16, ((const GLOBAL unsigned short*)p)[k]);
                acc = fma(x, x, acc);
            }
        }
    }
    return acc;
}

// Sums of squares in 64 bits, in a fixed order: one partial sum for each workgroup's elements.  One pass over the gradients, bound by
// memory: 89M fp32 in 55.5 us = 6.4 TB/s, 85M bf16 in 36 us = 4.7 TB/s (16 KB to 64 KB a workgroup: at most 8,192 partial sums is the
// best of 1,024 to 32,768: 86, 67, 61, 57, 60, 71 us for 120M bf16 values in 500 tensors when they took three launches; 50 us in
// two).  Eight loads in flight instead of four halve the occupancy (57 -> 60 us).
template <bool NT>
__global__ __launch_bounds__(256) void norm_partial_kernel(const OptTensors ts, double* __restrict__ partial)
{
    __shared__ double red[4];
    const Found f = find_part(ts, blockIdx.x);
    double acc = f.dt == 0 ? sum_squares<0, NT>(f.base, f.n) : f.dt == 1 ? sum_squares<1, NT>(f.base, f.n) : sum_squares<2, NT>(f.base, f.n);
    acc = wave_sum(acc);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = acc;
    __syncthreads();
    if (threadIdx.x == 0) partial[(size_t)ts.partial0 + blockIdx.x] = (red[0] + red[1]) + (red[2] + red[3]);
}

// adds the partial sums where no step does it itself: one workgroup, 2 us (one wave, up to 1,024 of them) or 4 us
__global__ __launch_bounds__(1024) void norm_final_kernel(const double* __restrict__ partial, uint32_t n, double max_norm,
                                                          float* __restrict__ norm_coef)
{
    __shared__ double red[16];
    if (n <= kOptWavePartials) {                             // (the order in which a step adds them)
        if (threadIdx.x >= 64) return;
        const NormCoef r = norm_coef_of(wave_total(partial, n), max_norm);
        if (threadIdx.x == 0) {
            norm_coef[0] = r.norm;
            norm_coef[1] = r.coef;
        }
        return;
    }
    double acc = 0.0;
    for (uint32_t i = threadIdx.x; i < n; i += 1024) acc += partial[i];
    acc = wave_sum(acc);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = acc;
    __syncthreads();
    if (threadIdx.x == 0) {
        double s = 0.0;
#pragma unroll
        for (int k = 0; k < 16; ++k) s += red[k];
        const NormCoef r = norm_coef_of(s, max_norm);
        norm_coef[0] = r.norm;
        norm_coef[1] = r.coef;
    }
}

// g *= *coef, rounded to nearest; a coefficient of 1 leaves the tensors alone.  Reads and writes the gradients once; the step that
// clips by itself does without.
__global__ __launch_bounds__(256) void scale_many_kernel(const OptTensors ts, const float* __restrict__ coef)
{
    const float c = *coef;
    if (c == 1.f) return;
    const Found f = find_part(ts, blockIdx.x);
    const uint32_t n = f.n;
    void* const q0 = (void*)f.base;
    for (uint32_t i = threadIdx.x * 4; i < n; i += 1024) {
        float g[4];
        if (f.dt == 0) load_elements<0, 4, false, false>(q0, i, n).values(g);
        else if (f.dt == 1) load_elements<1, 4, false, false>(q0, i, n).values(g);
        else load_elements<2, 4, false, false>(q0, i, n).values(g);
#pragma unroll
        for (int k = 0; k < 4; ++k) g[k] *= c;
        if (f.dt == 0) store_f32<4, false, false>(q0, i, n, g);
        else {
            unsigned short q[4];
#pragma unroll
            for (int k = 0; k < 4; ++k)
                q[k] = f.dt == 1 ? bf16_nearest(g[k]) : __builtin_bit_cast(unsigned short, (_Float16)g[k]);
            store_u16<4, false, false>(q0, i, n, q);
        }
    }
}

// ---- moments to 8 bits and back ----------------------------------------------------------------------------------------
// To the nearest: the stochastic rounding's cut with half a step added; values that 8 bits hold come back as they are.  One pass, 10
// bytes an element either way: 3.2M packed in 7.2 us (4.5 TB/s, the launch in it), 60M read back in 87 us = 6.9 TB/s.
__global__ __launch_bounds__(256) void moments_pack_kernel(const float* __restrict__ m, const float* __restrict__ v, uint64_t n,
                                                           uint8_t* __restrict__ m8, uint8_t* __restrict__ me, uint8_t* __restrict__ r8,
                                                           uint8_t* __restrict__ re)
{
    const uint64_t base = (uint64_t)blockIdx.x * 1024, left = n - base;
    const uint32_t nb = left < 1024 ? (uint32_t)left : 1024, i = threadIdx.x * 4;
    if (i >= round_up_block(nb)) return;
    float a[4], v4[4], b[4];
    const Elements<0, 4> qm = load_elements<0, 4, false, true>(m + base, i, nb), qv = load_elements<0, 4, false, true>(v + base, i, nb);
    qm.values(a);
    qv.values(v4);
    const bool plain = roots<4>(v4, b);
    const uint32_t em = block_scale<4, false>(a), er = block_scale<4, true>(b);
    const uint32_t half[4] = {0x80000000u, 0x80000000u, 0x80000000u, 0x80000000u};
    *(Codes<4>*)(m8 + base + i) = e4m3_codes<4>(a, em, half);
    *(Codes<4>*)(r8 + base + i) = e4m3_root_codes<4>(b, plain, er, half);
    if ((i & 31) == 0) {
        me[(base + i) / kOptBlock] = (uint8_t)(em >> 23);
        re[(base + i) / kOptBlock] = (uint8_t)(er >> 23);
    }
}

__global__ __launch_bounds__(256) void moments_unpack_kernel(const uint8_t* __restrict__ m8, const uint8_t* __restrict__ me,
                                                             const uint8_t* __restrict__ r8, const uint8_t* __restrict__ re,
                                                             float* __restrict__ m, float* __restrict__ v, uint64_t n)
{
    const uint64_t base = (uint64_t)blockIdx.x * 1024, left = n - base;
    const uint32_t nb = left < 1024 ? (uint32_t)left : 1024, i = threadIdx.x * 4;
    if (i >= nb) return;
    float a[4], b[4];
    e4m3_values<4>(*(const Codes<4>*)(m8 + base + i), me[(base + i) / kOptBlock], a);
    e4m3_values<4>(*(const Codes<4>*)(r8 + base + i), re[(base + i) / kOptBlock], b);
#pragma unroll
    for (int k = 0; k < 4; ++k) b[k] *= b[k];
    store_f32<4, false, true>(m + base, i, nb, a);
    store_f32<4, false, true>(v + base, i, nb, b);
}

}  // namespace

uint32_t opt_mix(uint32_t x) { return mix32(x); }

template <int BITS>
static void (*adamw_kernel_of(int list, bool streaming))(AdamWArgs)
{
    if (list == 0) return streaming ? adamw_many_kernel<BITS, 0, true> : adamw_many_kernel<BITS, 0, false>;
    if (list == 1) return streaming ? adamw_many_kernel<BITS, 1, true> : adamw_many_kernel<BITS, 1, false>;
    return streaming ? adamw_many_kernel<BITS, 2, true> : adamw_many_kernel<BITS, 2, false>;
}

hipError_t launch_adamw_many(const AdamWArgs& a, int bits, int list, bool streaming, uint32_t blocks, hipStream_t s)
{
    auto* k = bits == 32 ? adamw_kernel_of<32>(list, streaming) : adamw_kernel_of<8>(list, streaming);
    // Past the caches fewer workgroups at a time are faster: each has four streams that it reads and writes, and the fewer there are
    // the longer memory stays with one.  LDS that nobody uses keeps it at three to a CU.  Measured with 6 (8 for 32 bits) | 5 | 3 |
    // 2 a CU, us: 8 bits 100M fp32 parameters with clipping 373 | 360 | 356 | 379; 32 bits 268M fp32 1320 | 1308 | 1308 | 1297, 40M bf16
    // 164.5 | 162.3 | 161.6 | 158.6.  8 bits with bf16 parameters, where arithmetic takes the time, want all they can get: 268M
    // parameters 483 | 494 | 513 | 601.
    const unsigned idle_lds = streaming && !(bits == 8 && list == 1) ? 53000 : 0;
    hipLaunchKernelGGL(k, dim3(blocks), dim3(256), idle_lds, s, a);
    return hipGetLastError();
}

hipError_t launch_norm_partial(const OptTensors& ts, bool streaming, uint32_t blocks, double* partial, hipStream_t s)
{
    auto* k = streaming ? norm_partial_kernel<true> : norm_partial_kernel<false>;
    hipLaunchKernelGGL(k, dim3(blocks), dim3(256), 0, s, ts, partial);
    return hipGetLastError();
}

hipError_t launch_norm_final(const double* partial, uint32_t n, double max_norm, float* norm_coef, hipStream_t s)
{
    hipLaunchKernelGGL(norm_final_kernel, dim3(1), dim3(n <= kOptWavePartials ? 64 : 1024), 0, s, partial, n, max_norm, norm_coef);
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
