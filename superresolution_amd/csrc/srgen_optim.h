// srgen_optim.h -- kernel launch interface of the optimizer operators over many tensors (srgen_optim_api.cpp checks and
// batches, srgen_optim_kernels.hip computes).  Not part of the public ABI (include/srgen.h).
#pragma once
#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace srgen {

// Tensors travel to the kernels by value, in the kernel arguments (4 KiB at most): nothing is uploaded, nothing is kept
// between calls, and a captured graph holds its own copy.  An address has 48 bits and is even; descriptors use the other bits.
constexpr int kOptBlock = 32;        // elements that share one power-of-two scale (8-bit moments)
constexpr int kOptChunk = 4096;      // elements of one workgroup of the step, and of one step counter
constexpr int kOptMaxTensors = 320;  // tensors of one launch of the step
constexpr int kOptMaxListed = 336;   // ... of the norm and the scaling
constexpr uint32_t kOptMaxPart = 16384;      // most elements of one workgroup of those (the last one's count takes 14 bits)
constexpr uint32_t kOptWavePartials = 1024;  // partial sums that one wave adds (in the step's own workgroups: no launch between)
constexpr uint64_t kAddrMask = (1ull << 48) - 1;

// One chunk of a list that takes steps (the table is made once for a list: it depends on the sizes alone).
struct OptChunk {
    uint32_t tensor;       // in the list
    uint32_t index;        // of the chunk in its tensor
    uint32_t offset32;     // start in the moments' buffers, in blocks of 32 elements
    uint32_t count;        // elements, 1 .. kOptChunk
};

struct AdamWScalars {
    double beta1, beta2, ln_beta1, ln_beta2, lr, eps, wd;
    const float* lr_dev;
    const float* grad_mul;
    const float* grad_div;
    const float* found_inf;
    const double* partial; // partial sums of the gradients' squares, or NULL: the step clips by their norm
    double max_norm;
    float* norm_coef;      // {norm, coefficient}, written where partial is set
    uint32_t partials;     // 1 .. kOptWavePartials
    uint32_t seed_key;     // mix(seed)
    int negate;
};
struct MomentPtrs {
    void* m;               // fp32, or e4m3 codes
    void* v;               // fp32 second moment, or e4m3 codes of its square root
    uint8_t* m_scale;
    uint8_t* v_scale;
    int32_t* step;
    const OptChunk* chunks;
};
struct AdamWArgs {
    // addresses of parameters and gradients, the lowest bit set where the elements are bf16; gradient 0: the tensor takes no step
    uint32_t p[kOptMaxTensors], g[kOptMaxTensors];
    uint32_t hi[kOptMaxTensors];  // the parameter's upper 16 bits, the gradient's << 16
    uint32_t tensor0;             // the list's tensor that p[0], g[0] are of
    uint32_t chunk0;              // chunk (and step counter) of workgroup 0
    AdamWScalars sc;
    MomentPtrs mo;
};
static_assert(sizeof(AdamWArgs) <= 4096, "kernel arguments hold 4 KiB");

// a list without a table: each workgroup takes `part` elements of one tensor
struct OptTensors {
    uint64_t t[kOptMaxListed];              // address | type << 48 | (elements of its last workgroup - 1) << 50
    uint32_t block0[kOptMaxListed + 1];     // first workgroup of the tensor; behind the last tensor: their number
    uint32_t part;                          // a power of two up to kOptMaxPart
    int count;
    uint32_t partial0;                      // norm: partial sum of workgroup 0
};
static_assert(sizeof(OptTensors) <= 4096 - 24, "kernel arguments hold 4 KiB");

uint32_t opt_mix(uint32_t x);        // the hash of the stochastic rounding (host side, for the seed)

hipError_t launch_adamw_many(const AdamWArgs& a, int bits, int list, bool streaming, uint32_t blocks, hipStream_t s);
hipError_t launch_norm_partial(const OptTensors& ts, bool streaming, uint32_t blocks, double* partial, hipStream_t s);
hipError_t launch_norm_final(const double* partial, uint32_t n, double max_norm, float* norm_coef, hipStream_t s);
hipError_t launch_scale_many(const OptTensors& ts, uint32_t blocks, const float* coef, hipStream_t s);
hipError_t launch_moments_pack(const float* m, const float* v, size_t n, uint8_t* m8, uint8_t* me, uint8_t* r8, uint8_t* re,
                               hipStream_t s);
hipError_t launch_moments_unpack(const uint8_t* m8, const uint8_t* me, const uint8_t* r8, const uint8_t* re, float* m, float* v,
                                 size_t n, hipStream_t s);

}  // namespace srgen
