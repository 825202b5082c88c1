// linear_attention.cuh -- what the two kernels of linear attention share
// (linear_attention.cu, linear_attention_umma.cu): their parameters, and values as sums
// of bf16 ones.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace need {
namespace attention {

struct Stream {
    const void* p;
    int64_t sb, st, sh;  // element strides of sequence, token, head
    int32_t share;       // heads that share one of this tensor's
};

struct AttnParams {
    Stream q, k, v;
    const float* ld;
    int64_t lb, lt, lh;
    const uint8_t* seg;
    int64_t gb, gt;
    const float* s0;
    float* sT;
    void* out;
    int64_t ob, ot, oh;
    int64_t T;
    int32_t H, dk, dv, slices, nseg;
    int64_t first_chunks, seg_chunks;  // of 64 tokens: of the first segment of the sequence, of the others
    // The launch ahead runs all segments but the last for the state that they leave (from
    // none); the one after it runs them for their outputs.  lead: the first one's outputs come
    // ahead, and its state with them.
    int32_t ahead, lead;
    float scale;          // at most 2^32, so that no decay's product with it is past fp32
    float late;           // a larger one, of the outputs (scale is 1 then); else 1
    float* part;          // [chain, nseg - 1, dk, dv]: the segments' own states, then those that enter the next
    float* part_d;        // [chain, nseg - 1, 2]: their decays as products of two, below 0 where a reset lies in between
    const uint32_t* redo; // of each block, null for all: whether it has to run
    __host__ __device__ int launched() const { return ahead ? nseg - 1 : nseg - lead; }  // segments of this launch
    __host__ __device__ int64_t segment(int s) const { return s == 0 ? 0 : first_chunks + (s - 1) * seg_chunks; }  // its first chunk
};

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ float2 unpack_bf16(uint32_t u) {
    return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
}
__device__ __forceinline__ float2 splat(float x) { return make_float2(x, x); }
// The two of x as the sums of N bf16 values each.
template <int N>
__device__ __forceinline__ void split(float2 x, uint32_t (&pl)[N]) {
#pragma unroll
    for (int n = 0; n < N; ++n) {
        pl[n] = pack_bf16(x.x, x.y);
        if (n + 1 < N) {
            const float2 f = unpack_bf16(pl[n]);
            x = __ffma2_rn(f, splat(-1.0f), x);
        }
    }
}

// A segment's decay is the product of its chunks' in fp64, and kept as that of two floats: a growing one
// passes fp32's range before the states that it multiplies do.  Neither float is 0 or infinite, so that
// states of 0 and infinity stay.
__device__ __forceinline__ void put_decay(float* to, double d) {
    const bool plain = d == -1.0 || d != d;
    const int h = plain ? 0 : max(-252, min(252, ilogb(d))) >> 1;
    const float a = static_cast<float>(ldexp(d, -h));
    to[0] = plain ? a : fminf(fmaxf(a, 0x1p-126f), 0x1p126f), to[1] = ldexpf(1.0f, h);
}
// The state of a segment's start at its end.
__device__ __forceinline__ float times_state(float2 d, float s) { return d.x == -1.0f ? 0.0f : s * d.x * d.y; }

// Whether a segment starts at token t: the state before it is not read then, whatever it holds.
__device__ __forceinline__ bool starts(const float* ld, int64_t lt, const uint8_t* marks, int64_t gt, int64_t t) {
    return (marks != nullptr && marks[t * gt] != 0) || ld[t * lt] == -INFINITY;
}

// The kernel on the tensor cores of sm_100a (linear_attention_umma.cu): chunks of 128
// tokens, bf16, up to 128 features.  `redo` [blocks] tells which of attention_kernel's
// blocks it leaves to that.  state: only the segments' states.
bool umma_takes(const AttnParams& p, int64_t nb);
int umma_run(const AttnParams& p, int64_t nb, uint32_t* redo, cudaStream_t stream);

}  // namespace attention
}  // namespace need
