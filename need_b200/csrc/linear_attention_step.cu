// linear_attention_step.cu -- linear attention with a decay for each head, one token of
// each sequence (need_linear_attention_step):
//
//   S = a S + k^T v,   out = scale q S,   a = exp(log_decay)
//
// in fp32, the states in place in a pool.  The state is read and written once, 8 B per
// element: that is all the traffic that counts, so the kernel is bound by HBM.  A team of
// threads takes a (sequence, head, up to 128 columns): a thread owns 4 columns (16 bytes) of
// every R-th row, its rows' loads in flight together, and the row groups' parts of q S are
// added in a fixed order.  A CTA is 1 to 4 teams, heads of one sequence.  256 tokens of 13
// heads of 64 x 64: 15.4 us warm (in part from L2; 16.9 at HBM's rate); 128 of 32 of 128 x 128:
// 86 us, 6.3 TB/s.  With slots every CTA looks for its slot among those before it, which
// 4096 tokens of 8 heads show: 158 us without, 185 with.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <type_traits>

#include "host_common.h"
#include "need_scan.h"

using namespace need;

namespace {

constexpr int kThreads = 128, kMaxThreads = 512, kCols = 128;  // columns of a team
constexpr int kRows = 8;                                          // of a thread in flight

struct StepParams {
    need_heads q, k, v;
    const float* ld;
    int64_t ln, lh;
    float* state;
    int64_t ss, slots;
    const int32_t* slot;
    void* out;
    int64_t on, oh;
    int32_t H, dk, dv, groups;  // groups: of a team's columns, a power of two
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
// TEAMS of a CTA.
template <typename T, bool VEC, int TEAMS>
__global__ void __launch_bounds__(TEAMS == 1 ? kMaxThreads : kThreads) step_kernel(const StepParams p) {
    constexpr int W = VEC ? 4 : 1, B = kRows;  // columns of a thread
    extern __shared__ float smem[];        // of each team k, q, then the row groups' sums
    const int threads = TEAMS == 1 ? blockDim.x : kThreads / TEAMS;
    const int tid = TEAMS == 1 ? threadIdx.x : threadIdx.x % (kThreads / TEAMS), team = TEAMS == 1 ? 0 : threadIdx.x / (kThreads / TEAMS);
    const int per = (p.H + TEAMS - 1) / TEAMS;  // CTAs of a sequence
    const int64_t n = blockIdx.x / per;
    const int h0 = static_cast<int>(blockIdx.x % per) * TEAMS + team, h = TEAMS == 1 || h0 < p.H ? h0 : p.H - 1;
    float* const sh = smem + team * (2 * p.dk + threads * W);
    const int rows = threads / p.groups, r0 = tid / p.groups, j = blockIdx.y * (p.groups * W) + (tid % p.groups) * W;
    const bool mine = (TEAMS == 1 || h0 < p.H) && j < p.dv;
    const int64_t where = p.slot != nullptr ? p.slot[n] : n;
    T* const out = static_cast<T*>(p.out) + n * p.on + h * p.oh;
    bool taken = where >= p.slots;
    if (p.slot != nullptr && where >= 0)
        for (int64_t m = threadIdx.x; m < n; m += blockDim.x) taken |= p.slot[m] == where;
    const T *k = row_of<T>(p.k, n, h, p.H), *q = row_of<T>(p.q, n, h, p.H), *v = row_of<T>(p.v, n, h, p.H);
    const float x = p.ld[n * p.ln + h * p.lh];
    float* const s = p.state + where * p.ss + h * (int64_t(p.dk) * p.dv) + j;
    float vj[W], o[W], u[B][W];
    auto load = [&](int i0) {
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
    };
    if (where >= 0 && where < p.slots) load(r0);  // not kept where the slot turns out to be taken
#pragma unroll
    for (int e = 0; e < W; ++e) vj[e] = mine ? to_float(v[j + e]) : 0.0f, o[e] = 0.0f;
    for (int i = tid; i < p.dk; i += threads) sh[i] = to_float(k[i]), sh[p.dk + i] = to_float(q[i]);
    if (__syncthreads_or(taken) || where < 0) {
        if (r0 == 0)
            for (int e = 0; e < W; ++e)
                if (mine) out[j + e] = static_cast<T>(where < 0 ? 0.0f : __int_as_float(0x7fc00000));
        return;
    }
    const bool reset = x == -INFINITY;
    const float a = expf(x);
    for (int i0 = r0; i0 < p.dk; i0 += rows * B) {
        if (i0 != r0) load(i0);
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
    for (int c = tid; c < cols; c += threads) {
        const int jc = blockIdx.y * cols + c;
        if (jc >= p.dv || (TEAMS > 1 && h0 >= p.H)) break;
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
    if (a->log_decay == nullptr || (a->state == nullptr && a->slots > 0) || a->out == nullptr)
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
    // Where the threads of all states fit the GPU at once, a state's rows are in flight at
    // once (3 of 8 heads of 128 x 96 in fp16 take 512 threads each 4.7 us, 128 each 6.7;
    // but 16 of 32 of 128 x 128 15.9 and 9.8).  Small states share a CTA.
    const int64_t states = a->n * a->H, rows = (a->dk + kRows - 1) / kRows;  // threads that a column group can use
    int threads = kThreads;
    while (threads < kMaxThreads && threads < p.groups * rows && states * threads * 2 <= 148 * kMaxThreads) threads *= 2;
    int teams = 1;
    while (teams < 4 && teams < a->H && threads == kThreads && threads / teams / 2 >= std::max<int64_t>(32, p.groups * rows)) teams *= 2;
    const int64_t cols = int64_t(p.groups) * w, tiles = (a->dv + cols - 1) / cols;
    if (tiles > 65535) return fail(NEED_ERR_UNSUPPORTED, "linear attention step: dv out of range");
    const dim3 grid(static_cast<unsigned>(a->n * ((a->H + teams - 1) / teams)), static_cast<unsigned>(tiles));
    const size_t bytes = (teams * 2 * a->dk + threads * w) * sizeof(float);
    auto go = [&](auto tag) {
        using T = decltype(tag);
        auto launch = [&](auto v) {
            constexpr bool V = decltype(v)::value;
            if (teams == 1) step_kernel<T, V, 1><<<grid, threads, bytes, stream>>>(p);
            else if (teams == 2) step_kernel<T, V, 2><<<grid, threads, bytes, stream>>>(p);
            else step_kernel<T, V, 4><<<grid, threads, bytes, stream>>>(p);
        };
        if (vec) launch(std::true_type{});
        else launch(std::false_type{});
    };
    if (a->dtype == NEED_F32) go(float{});
    else if (a->dtype == NEED_BF16) go(__nv_bfloat16{});
    else go(__half{});
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? ok() : cuda_fail(e, "linear attention step launch");
}
