// srgen_optim_api.cpp -- C ABI of the optimizer operators over a list of tensors (include/srgen.h): argument checks, and the
// list cut into launches whose descriptors fit the kernel arguments.
#include "../../include/srgen.h"
#include "srgen_internal.h"
#include "srgen_optim.h"

#include <math.h>

using namespace srgen;

static_assert(sizeof(OptChunk) == 16, "a table entry is four words");
static_assert(SRGEN_OPT_BLOCK == kOptBlock && SRGEN_OPT_CHUNK == kOptChunk, "include/srgen.h states the kernels' sizes");

namespace {

#define HIP_TRY(expr)                                                                      \
    do {                                                                                   \
        hipError_t e_ = (expr);                                                            \
        if (e_ != hipSuccess)                                                              \
            return fail(SRGEN_E_HIP, "%s failed: %s (%s:%d)", #expr, hipGetErrorString(e_), \
                        __FILE__, __LINE__);                                               \
    } while (0)

// workgroups of 256 threads in one launch: the grid is counted in threads, in 32 bits
constexpr uint64_t kMaxBlocks = (1ull << 24) - 1;

// What a step touches (parameters, gradients, moments) is still in the 256 MB Infinity Cache at the next one, or was written by the
// backward pass just now, unless it is larger than that: then loads and stores are marked non-temporal.  Measured, us without |
// with: 32 bits fp32 20M parameters (320 MB) 93 | 105, 24M (384 MB) 135 | 126; bf16 24M (288 MB) 84 | 98, 32M (384 MB) 140 | 129;
// 8 bits fp32 32M (322 MB) 87 | 91, 48M (483 MB) 151 | 135.
constexpr uint64_t kStreamingBytes = 350ull << 20;
// The norm only reads: 64 MB 14.4 | 12.7, 128 MB 24.4 | 22.8, 400 MB 74 | 65; but a step behind it finds small gradients in cache
// (3M parameters with clipping 24 | 27).
constexpr uint64_t kStreamingNormBytes = 128ull << 20;

inline size_t element_bytes(int dtype) { return dtype == SRGEN_F32 ? 4 : 2; }
inline bool aligned(const void* p, size_t a) { return ((uintptr_t)p & (a - 1)) == 0; }
inline uint64_t chunks_of(uint64_t n, uint64_t per) { return (n + per - 1) / per; }

int check_list(int count, const void* const* t, const uint64_t* numel, const int32_t* dtype, const char* what, bool f16)
{
    if (count < 0) return fail(SRGEN_E_INVALID, "count %d", count);
    if (count && (!t || !numel || !dtype)) return fail(SRGEN_E_INVALID, "NULL list");
    for (int i = 0; i < count; ++i) {
        if (numel[i] > kMaxBlocks * kOptChunk) return fail(SRGEN_E_UNSUPPORTED, "%s %d: %llu elements", what, i, (unsigned long long)numel[i]);
        if (dtype[i] != SRGEN_F32 && dtype[i] != SRGEN_BF16 && !(f16 && dtype[i] == SRGEN_F16))
            return fail(SRGEN_E_UNSUPPORTED, "%s %d: type %d", what, i, dtype[i]);
        if ((uintptr_t)t[i] > kAddrMask) return fail(SRGEN_E_UNSUPPORTED, "%s %d: an address of more than 48 bits", what, i);
        if (t[i] && !aligned(t[i], element_bytes(dtype[i]))) return fail(SRGEN_E_INVALID, "%s %d is not aligned to its element", what, i);
    }
    return SRGEN_OK;
}

// elements of one workgroup of the norm: more for long lists, so that the partial sums stay few
uint32_t norm_part(int count, const uint64_t* numel)
{
    uint64_t total = 0;
    for (int i = 0; i < count; ++i) total += numel[i];
    uint32_t per = kOptChunk;
    while (per < kOptMaxPart && total / per > 8192) per *= 2;
    return per;
}

// takes tensors from *i on into one launch, until its descriptors or its workgroups are full; the number of its workgroups
uint32_t fill_list(int count, const void* const* t, const uint64_t* numel, const int32_t* dtype, int* i, OptTensors* ts)
{
    uint64_t blocks = 0;
    ts->count = 0;
    for (; *i < count && ts->count < kOptMaxListed; ++*i) {
        const uint64_t n = t[*i] ? numel[*i] : 0, c = chunks_of(n, ts->part);
        if (blocks + c > kMaxBlocks) break;
        if (!c) continue;
        ts->t[ts->count] = (uint64_t)(uintptr_t)t[*i] | (uint64_t)dtype[*i] << 48 | (n - (c - 1) * ts->part - 1) << 50;
        ts->block0[ts->count++] = (uint32_t)blocks;
        blocks += c;
    }
    ts->block0[ts->count] = (uint32_t)blocks;
    return (uint32_t)blocks;
}

// the partial sums of the list's squares (tensors with g[i] == NULL are left out); the list has been checked
int norm_partials(int count, const void* const* g, const uint64_t* numel, const int32_t* dtype, const float* norm_coef2, void* scratch,
                  size_t scratch_bytes, void* stream, uint32_t* partials)
{
    if (!norm_coef2 || !aligned(norm_coef2, 4)) return fail(SRGEN_E_INVALID, "norm_coef2 is NULL or misaligned");
    const uint32_t per = norm_part(count, numel);
    uint64_t total = 0, bytes = 0;
    for (int i = 0; i < count; ++i) {
        if (!g[i]) continue;
        total += chunks_of(numel[i], per);
        bytes += numel[i] * element_bytes(dtype[i]);
    }
    if (total > 0xFFFFFFFFull) return fail(SRGEN_E_UNSUPPORTED, "%llu partial sums", (unsigned long long)total);
    if (total && (!scratch || !aligned(scratch, 8))) return fail(SRGEN_E_INVALID, "scratch is NULL or misaligned");
    if (scratch_bytes < total * sizeof(double))
        return fail(SRGEN_E_WORKSPACE, "scratch of %zu bytes, %zu needed", scratch_bytes, (size_t)total * sizeof(double));
    OptTensors ts;
    ts.part = per;
    ts.partial0 = 0;
    for (int i = 0; i < count;) {
        const uint32_t blocks = fill_list(count, g, numel, dtype, &i, &ts);
        if (blocks) HIP_TRY(launch_norm_partial(ts, bytes > kStreamingNormBytes, blocks, (double*)scratch, (hipStream_t)stream));
        ts.partial0 += blocks;
    }
    *partials = (uint32_t)total;
    return SRGEN_OK;
}

}  // namespace

extern "C" {

int srgen_adamw_chunk_count(int count, const uint64_t* numel, uint64_t* chunks)
{
    if (count < 0 || (count && !numel) || !chunks) return fail(SRGEN_E_INVALID, "NULL argument or count %d", count);
    uint64_t n = 0;
    for (int i = 0; i < count; ++i) n += chunks_of(numel[i], kOptChunk);
    *chunks = n;
    return SRGEN_OK;
}

int srgen_adamw_chunk_table(int count, const uint64_t* numel, const uint64_t* offset, uint32_t* host_table, uint64_t chunks)
{
    if (count < 0 || (count && (!numel || !offset)) || (chunks && !host_table)) return fail(SRGEN_E_INVALID, "NULL argument or count %d", count);
    uint64_t k = 0;
    for (int i = 0; i < count; ++i) {
        const uint64_t c = chunks_of(numel[i], kOptChunk);
        if (offset[i] % kOptBlock || (offset[i] + numel[i]) / kOptBlock > 0xFFFFFFFEull) return fail(SRGEN_E_INVALID, "offset %d: %llu", i, (unsigned long long)offset[i]);
        if (k + c > chunks) return fail(SRGEN_E_INVALID, "a table of %llu chunks is too short", (unsigned long long)chunks);
        for (uint64_t x = 0; x < c; ++x, ++k) {
            const uint64_t rest = numel[i] - x * kOptChunk;
            host_table[4 * k] = (uint32_t)i;
            host_table[4 * k + 1] = (uint32_t)x;
            host_table[4 * k + 2] = (uint32_t)(offset[i] / kOptBlock + x * (kOptChunk / kOptBlock));
            host_table[4 * k + 3] = (uint32_t)(rest < (uint64_t)kOptChunk ? rest : kOptChunk);
        }
    }
    return SRGEN_OK;
}

int srgen_adamw_many(int count, void* const* p, const void* const* g, const uint64_t* numel, const uint64_t* offset,
                     const int32_t* p_dtype, const int32_t* g_dtype, const srgen_moments* mo, const srgen_adamw_args* args, void* stream)
{
    if (int rc = check_list(count, p, numel, p_dtype, "parameter", false)) return rc;
    if (int rc = check_list(count, g, numel, g_dtype, "gradient", false)) return rc;
    if (!mo || !args || (count && !offset)) return fail(SRGEN_E_INVALID, "NULL argument");
    if (mo->bits != 8 && mo->bits != 32) return fail(SRGEN_E_UNSUPPORTED, "moments of %d bits: 8 or 32", mo->bits);
    // (not (x >= 0): NaN is refused as well)
    if (!(args->lr >= 0.0) || !(args->eps >= 0.0) || !(args->weight_decay >= 0.0) || !(args->beta1 >= 0.0 && args->beta1 < 1.0) ||
        !(args->beta2 >= 0.0 && args->beta2 < 1.0))
        return fail(SRGEN_E_INVALID, "lr %g, betas %g %g, eps %g, weight decay %g", args->lr, args->beta1, args->beta2, args->eps, args->weight_decay);
    uint64_t chunks = 0, step_bytes = 0;
    unsigned types = 0;                                    // bit 0: some fp32, bit 1: some bf16
    for (int i = 0; i < count; ++i) {
        if (g[i]) types |= 1u << p_dtype[i] | 1u << g_dtype[i];
        if (g[i]) step_bytes += numel[i] * (element_bytes(p_dtype[i]) + element_bytes(g_dtype[i]) + (mo->bits == 32 ? 8 : 2));
        if (numel[i] && !p[i]) return fail(SRGEN_E_INVALID, "parameter %d is NULL", i);
        if (offset[i] % kOptBlock || offset[i] / kOptBlock > 0xFFFFFFFFull) return fail(SRGEN_E_INVALID, "offset %d: %llu", i, (unsigned long long)offset[i]);
        if (offset[i] + chunks_of(numel[i], kOptBlock) * kOptBlock > mo->numel)
            return fail(SRGEN_E_INVALID, "the moments of tensor %d end behind their buffer", i);
        chunks += chunks_of(numel[i], kOptChunk);
    }
    if (chunks != mo->chunks) return fail(SRGEN_E_INVALID, "moments of %llu chunks, the list has %llu", (unsigned long long)mo->chunks, (unsigned long long)chunks);
    if (args->norm_coef2) {
        if (args->grad_mul) return fail(SRGEN_E_INVALID, "grad_mul and norm_coef2: one of the two");
        if (!(args->max_norm > 0.0)) return fail(SRGEN_E_INVALID, "max_norm %g", args->max_norm);
    }
    const size_t al = mo->bits == 32 ? 16 : 4;
    if (chunks && (!mo->m || !mo->v || !mo->step || !mo->table || (mo->bits == 8 && (!mo->m_scale || !mo->v_scale)))) return fail(SRGEN_E_INVALID, "NULL moments");
    if (!aligned(mo->m, al) || !aligned(mo->v, al) || !aligned(mo->step, 4) || !aligned(mo->table, 16)) return fail(SRGEN_E_INVALID, "misaligned moments");

    const float* mul = args->grad_mul;
    const double* partial = nullptr;
    uint32_t partials = 0;
    if (args->norm_coef2) {
        if (int rc = norm_partials(count, g, numel, g_dtype, args->norm_coef2, args->norm_scratch, args->norm_scratch_bytes, stream, &partials)) return rc;
        // (found_inf may end the step's workgroups before they add anything, and the norm is wanted all the same)
        if (partials && partials <= kOptWavePartials && !args->found_inf) partial = (const double*)args->norm_scratch;
        else {
            HIP_TRY(launch_norm_final((const double*)args->norm_scratch, partials, args->max_norm, args->norm_coef2, (hipStream_t)stream));
            mul = args->norm_coef2 + 1;
        }
    }
    if (!chunks) return SRGEN_OK;
    AdamWArgs a;
    a.sc = AdamWScalars{args->beta1, args->beta2, log(args->beta1), log(args->beta2), args->lr, args->eps, args->weight_decay, args->lr_dev,
                        mul, args->grad_div, args->found_inf, partial, args->max_norm, args->norm_coef2, partials, opt_mix(args->seed),
                        args->maximize};
    a.mo = MomentPtrs{mo->m, mo->v, mo->m_scale, mo->v_scale, mo->step, reinterpret_cast<const OptChunk*>(mo->table)};
    const bool streaming = step_bytes > kStreamingBytes;
    uint64_t done = 0;                                     // chunks of the launches so far
    for (int i = 0; i < count;) {
        uint64_t blocks = 0;
        int k = 0;
        bool any = false;
        a.tensor0 = (uint32_t)i;
        for (; i < count && k < kOptMaxTensors; ++i, ++k) {
            const uint64_t c = chunks_of(numel[i], kOptChunk);
            if (blocks + c > kMaxBlocks) break;
            const uint64_t pa = (uint64_t)(uintptr_t)p[i] | (p_dtype[i] == SRGEN_BF16);
            const uint64_t ga = g[i] ? (uint64_t)(uintptr_t)g[i] | (g_dtype[i] == SRGEN_BF16) : 0;
            a.p[k] = (uint32_t)pa;
            a.g[k] = (uint32_t)ga;
            a.hi[k] = (uint32_t)(pa >> 32) | (uint32_t)(ga >> 32) << 16;
            any |= g[i] && c;
            blocks += c;
        }
        a.chunk0 = (uint32_t)done;
        done += blocks;
        if (any) HIP_TRY(launch_adamw_many(a, mo->bits, types == 1 ? 0 : types == 2 ? 1 : 2, streaming, (uint32_t)blocks, (hipStream_t)stream));
    }
    return SRGEN_OK;
}

int srgen_total_norm_scratch_bytes(int count, const uint64_t* numel, size_t* bytes)
{
    if (count < 0 || (count && !numel) || !bytes) return fail(SRGEN_E_INVALID, "NULL argument or count %d", count);
    const uint32_t per = norm_part(count, numel);
    uint64_t n = 0;
    for (int i = 0; i < count; ++i) n += chunks_of(numel[i], per);
    *bytes = (size_t)((n * sizeof(double) + 255) & ~(uint64_t)255);
    return SRGEN_OK;
}

int srgen_total_norm(int count, const void* const* g, const uint64_t* numel, const int32_t* dtype, double max_norm, float* norm_coef2,
                     void* scratch, size_t scratch_bytes, void* stream)
{
    if (int rc = check_list(count, g, numel, dtype, "tensor", true)) return rc;
    uint32_t partials = 0;
    if (int rc = norm_partials(count, g, numel, dtype, norm_coef2, scratch, scratch_bytes, stream, &partials)) return rc;
    HIP_TRY(launch_norm_final((const double*)scratch, partials, max_norm, norm_coef2, (hipStream_t)stream));
    return SRGEN_OK;
}

int srgen_scale_many(int count, void* const* g, const uint64_t* numel, const int32_t* dtype, const float* coef, void* stream)
{
    if (int rc = check_list(count, g, numel, dtype, "tensor", true)) return rc;
    if (!coef) return fail(SRGEN_E_INVALID, "coef is NULL");
    for (int i = 0; i < count; ++i)
        if (numel[i] && !g[i]) return fail(SRGEN_E_INVALID, "tensor %d is NULL", i);
    OptTensors ts;
    ts.part = kOptChunk;
    ts.partial0 = 0;
    for (int i = 0; i < count;) {
        const uint32_t blocks = fill_list(count, g, numel, dtype, &i, &ts);
        if (blocks) HIP_TRY(launch_scale_many(ts, blocks, coef, (hipStream_t)stream));
    }
    return SRGEN_OK;
}

static int check_pack(const void* m, const void* v, size_t n, const void* m8, const void* me, const void* r8, const void* re)
{
    if (!m || !v || !m8 || !me || !r8 || !re) return fail(SRGEN_E_INVALID, "NULL argument");
    if (!aligned(m, 4) || !aligned(v, 4) || !aligned(m8, 4) || !aligned(r8, 4)) return fail(SRGEN_E_INVALID, "operands must be 4-byte aligned");
    if (n > kMaxBlocks * 1024) return fail(SRGEN_E_UNSUPPORTED, "%zu elements", n);
    return SRGEN_OK;
}

int srgen_moments_pack(const float* m, const float* v, size_t numel, uint8_t* m8, uint8_t* me, uint8_t* r8, uint8_t* re, void* stream)
{
    if (numel == 0) return SRGEN_OK;
    if (int rc = check_pack(m, v, numel, m8, me, r8, re)) return rc;
    HIP_TRY(launch_moments_pack(m, v, numel, m8, me, r8, re, (hipStream_t)stream));
    return SRGEN_OK;
}

int srgen_moments_unpack(const uint8_t* m8, const uint8_t* me, const uint8_t* r8, const uint8_t* re, float* m, float* v, size_t numel,
                         void* stream)
{
    if (numel == 0) return SRGEN_OK;
    if (int rc = check_pack(m, v, numel, m8, me, r8, re)) return rc;
    HIP_TRY(launch_moments_unpack(m8, me, r8, re, m, v, numel, (hipStream_t)stream));
    return SRGEN_OK;
}

}  // extern "C"
