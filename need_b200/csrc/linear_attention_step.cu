// linear_attention_step.cu -- linear attention with a decay for each head, one token of
// each sequence (need_linear_attention_step):
//
//   S = a S + k^T v,   out = scale q S,   a = exp(log_decay)
//
// in fp32, the states in place in a pool.  The state is read and written once, 8 B per
// element: that is all the traffic that counts, so the kernel is bound by HBM.  One CTA
// per (sequence, head, up to 128 columns): a thread owns 4 columns (16 bytes) of every
// R-th row, its rows' loads in flight together, and the row groups' parts of q S are added
// in a fixed order.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "host_common.h"
#include "need_scan.h"

using namespace need;

namespace {

constexpr int kThreads = 128, kCols = 128;  // columns of a CTA

struct StepParams {
    need_heads q, k, v;
    const float* ld;
    int64_t ln, lh;
    float* state;
    int64_t ss, slots;
    const int32_t* slot;
    void* out;
    int64_t on, oh;
    int32_t H, dk, dv, groups;  // groups: of columns in a CTA, a power of two
    float scale;
};

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }

template <typename T>
__device__ __forceinline__ const T* row_of(const need_heads& x, int64_t n, int h, int H) {
    return static_cast<const T*>(x.ptr) + n * x.stride_b + (h / (H / static_cast<int>(x.heads))) * x.stride_h;
}

// VEC: rows of the state in whole, aligned groups of 4 columns; else a thread owns one.
template <typename T, bool VEC>
__global__ void __launch_bounds__(kThreads) step_kernel(const StepParams p) {
    constexpr int W = VEC ? 4 : 1, B = 8;  // columns of a thread, rows in flight
    extern __shared__ float sh[];          // k, q, then the row groups' sums
    const int64_t n = blockIdx.x / p.H;
    const int h = static_cast<int>(blockIdx.x % p.H), tid = threadIdx.x;
    const int rows = kThreads / p.groups, r0 = tid / p.groups, j = blockIdx.y * (p.groups * W) + (tid % p.groups) * W;
    const bool mine = j < p.dv;
    const int64_t where = p.slot != nullptr ? p.slot[n] : n;
    T* const out = static_cast<T*>(p.out) + n * p.on + h * p.oh;
    bool taken = where >= p.slots;
    if (p.slot != nullptr && where >= 0)
        for (int64_t m = tid; m < n; m += kThreads) taken |= p.slot[m] == where;
    const T *k = row_of<T>(p.k, n, h, p.H), *q = row_of<T>(p.q, n, h, p.H), *v = row_of<T>(p.v, n, h, p.H);
    for (int i = tid; i < p.dk; i += kThreads) sh[i] = to_float(k[i]), sh[p.dk + i] = to_float(q[i]);
    if (__syncthreads_or(taken) || where < 0) {
        if (r0 == 0)
            for (int e = 0; e < W; ++e)
                if (mine) out[j + e] = static_cast<T>(where < 0 ? 0.0f : __int_as_float(0x7fc00000));
        return;
    }
    const float x = p.ld[n * p.ln + h * p.lh];
    const bool reset = x == -INFINITY;
    const float a = expf(x);
    float* const s = p.state + where * p.ss + h * (int64_t(p.dk) * p.dv) + j;
    float vj[W], o[W];
#pragma unroll
    for (int e = 0; e < W; ++e) vj[e] = mine ? to_float(v[j + e]) : 0.0f, o[e] = 0.0f;
    for (int i0 = r0; i0 < p.dk; i0 += rows * B) {
        float u[B][W];
#pragma unroll
        for (int b = 0; b < B; ++b) {
            const int i = i0 + b * rows;
            if (mine && i < p.dk) {
                if constexpr (VEC) {
                    const float4 f = __ldcs(reinterpret_cast<const float4*>(s + int64_t(i) * p.dv));
                    u[b][0] = f.x, u[b][1] = f.y, u[b][2] = f.z, u[b][3] = f.w;
                } else {
                    u[b][0] = s[int64_t(i) * p.dv];
                }
            }
        }
#pragma unroll
        for (int b = 0; b < B; ++b) {
            const int i = i0 + b * rows;
            if (mine && i < p.dk) {
                const float kk = sh[i], qq = sh[p.dk + i];
#pragma unroll
                for (int e = 0; e < W; ++e) {
                    u[b][e] = reset ? kk * vj[e] : fmaf(a, u[b][e], kk * vj[e]);
                    o[e] = fmaf(qq, u[b][e], o[e]);
                }
                if constexpr (VEC) __stcs(reinterpret_cast<float4*>(s + int64_t(i) * p.dv), make_float4(u[b][0], u[b][1], u[b][2], u[b][3]));
                else s[int64_t(i) * p.dv] = u[b][0];
            }
        }
    }
    float* const red = sh + 2 * p.dk;
#pragma unroll
    for (int e = 0; e < W; ++e) red[(r0 * p.groups + tid % p.groups) * W + e] = o[e];
    __syncthreads();
    const int cols = p.groups * W;
    for (int c = tid; c < cols; c += kThreads) {
        const int jc = blockIdx.y * cols + c;
        if (jc >= p.dv) break;
        float sum = 0.0f;
        for (int r = 0; r < rows; ++r) sum += red[r * cols + c];
        out[jc] = static_cast<T>(p.scale * sum);
    }
}

}  // namespace

extern "C" int need_linear_attention_step(const need_linear_attention_step_args* a, need_stream_t stream) {
    if (a == nullptr) return fail(NEED_ERR_INVALID, "linear attention step: args is null");
    if (!dtype_ok(a->dtype)) return fail(NEED_ERR_UNSUPPORTED, "linear attention step: dtype %d", a->dtype);
    if (a->n < 1 || a->H < 1 || a->dk < 1 || a->dv < 1 || a->slots < 0)
        return fail(NEED_ERR_INVALID, "linear attention step: sizes must be positive");
    if (a->dk > 2048 || a->dv > (1 << 20) || a->H > (1 << 24) || a->n > (int64_t(1) << 30) / a->H)
        return fail(NEED_ERR_UNSUPPORTED, "linear attention step: at most 2048 features a head (got %lld), sizes out of range",
                    static_cast<long long>(a->dk));
    for (const need_heads* x : {&a->q, &a->k, &a->v}) {
        if (x->ptr == nullptr) return fail(NEED_ERR_INVALID, "linear attention step: an input is null");
        if (x->heads < 1 || a->H % x->heads != 0)
            return fail(NEED_ERR_INVALID, "linear attention step: heads must divide H = %lld", static_cast<long long>(a->H));
    }
    if (a->log_decay == nullptr || a->state == nullptr || a->out == nullptr)
        return fail(NEED_ERR_INVALID, "linear attention step: log_decay, state and out are required");
    if (a->slot == nullptr && a->slots < a->n) return fail(NEED_ERR_INVALID, "linear attention step: fewer states than tokens");
    if (a->slots > 1 && a->state_stride < a->H * a->dk * a->dv)
        return fail(NEED_ERR_INVALID, "linear attention step: the states overlap");
    StepParams p{};
    p.q = a->q, p.k = a->k, p.v = a->v, p.ld = a->log_decay, p.ln = a->ld_stride_n, p.lh = a->ld_stride_h;
    p.state = a->state, p.ss = a->state_stride, p.slots = a->slots, p.slot = a->slot;
    p.out = a->out, p.on = a->out_stride_n, p.oh = a->out_stride_h;
    p.H = int32_t(a->H), p.dk = int32_t(a->dk), p.dv = int32_t(a->dv), p.scale = a->scale;
    const bool vec = a->dv % 4 == 0 && aligned16(a->state) && (a->slots <= 1 || a->state_stride % 4 == 0);
    const int w = vec ? 4 : 1;
    const int64_t need = (std::min<int64_t>(a->dv, kCols) + w - 1) / w;
    p.groups = 1;
    while (p.groups < need) p.groups *= 2;
    const int64_t cols = int64_t(p.groups) * w, tiles = (a->dv + cols - 1) / cols;
    if (tiles > 65535) return fail(NEED_ERR_UNSUPPORTED, "linear attention step: dv out of range");
    const dim3 grid(static_cast<unsigned>(a->n * a->H), static_cast<unsigned>(tiles));
    const size_t bytes = (2 * a->dk + kThreads * w) * sizeof(float);
    auto go = [&](auto tag) {
        using T = decltype(tag);
        if (vec) step_kernel<T, true><<<grid, kThreads, bytes, stream>>>(p);
        else step_kernel<T, false><<<grid, kThreads, bytes, stream>>>(p);
    };
    if (a->dtype == NEED_F32) go(float{});
    else if (a->dtype == NEED_BF16) go(__nv_bfloat16{});
    else go(__half{});
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? ok() : cuda_fail(e, "linear attention step launch");
}
