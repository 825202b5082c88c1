// train_conv.cu -- the SSD block's causal depthwise conv + SiLU with its
// gradient (need_conv_silu_train_forward, need_conv_silu_train_backward).
//
//   v_t = bias + sum_d w[K-1-d] u_{t-d}  (u_{t-d} in t's segment), y = v s(v)
//   dv = dy s(v) (1 + v s(-v));  du_t = sum_d w[K-1-d] dv_{t+d}  (t+d in t's segment)
//   dw[K-1-d] = sum over b, t of dv_t u_{t-d};  dbias = sum of dv
//
// All in fp32, rounded once on the way out.  Bound by HBM (4 B per 16-bit
// element forward, 6 B backward): a thread walks kTok tokens of 4 channels
// (8- or 16-byte loads, kAhead rows in flight), with the last K-1 inputs, and
// backward the K-1 unfinished du, in registers; v is computed again rather
// than kept.  The backward reads the K-1 rows behind its tokens a second time
// (L2) for the dv they need.  A thread's sums for dw and dbias are added over
// the block's token ranges in shared memory, and column_sums adds the blocks'
// rows in a fixed order.
#include "host_common.h"
#include "need_scan.h"
#include "scan_kernel.cuh"
#include "train_common.cuh"

using namespace need;

namespace {

constexpr int kMaxTaps = 4;
constexpr int kTok = 32;     // tokens per thread
constexpr int kAhead = 4;    // rows loaded together
constexpr int kRanges = 4;   // token ranges per block (threadIdx.y)

struct ConvTrainParams {
    const void* u;
    int64_t usb, ust;
    const float* w;
    const float* bias;
    const uint8_t* seg;
    int64_t sgb, sgt;
    const void* gout;
    int64_t gsb, gst;
    void* out;    // y, or du
    float* part;  // [nb * ntb, C * (K + 1)]
    int32_t nb, T, C, ncg, ntb;  // channel groups (of 128) and token blocks
};

template <typename T>
__device__ __forceinline__ void load4(const T* p, float2 (&f)[2]) {
    if constexpr (Ops<T>::BYTES == 4) {
        const float4 v = *reinterpret_cast<const float4*>(p);
        f[0] = make_float2(v.x, v.y);
        f[1] = make_float2(v.z, v.w);
    } else {
        const uint2 v = *reinterpret_cast<const uint2*>(p);
        f[0] = widen(*reinterpret_cast<const typename Ops<T>::P*>(&v.x));
        f[1] = widen(*reinterpret_cast<const typename Ops<T>::P*>(&v.y));
    }
}
template <typename T>
__device__ __forceinline__ void store4(T* p, const float2 (&f)[2]) {
    typename Ops<T>::P h[2] = {Ops<T>::pack(f[0].x, f[0].y), Ops<T>::pack(f[1].x, f[1].y)};
    if constexpr (Ops<T>::BYTES == 4) *reinterpret_cast<float4*>(p) = *reinterpret_cast<const float4*>(h);
    else *reinterpret_cast<uint2*>(p) = *reinterpret_cast<const uint2*>(h);
}

template <typename T, int K, bool BWD>
__global__ void __launch_bounds__(32 * kRanges) conv_train_kernel(const ConvTrainParams p) {
    constexpr int H = K > 1 ? K - 1 : 1;
    const int cg = blockIdx.x % p.ncg;
    const int rest = blockIdx.x / p.ncg;
    const int tb = rest % p.ntb, b = rest / p.ntb;
    const int c0 = cg * 128 + threadIdx.x * 4;
    const int64_t tfirst = (int64_t(tb) * kRanges + threadIdx.y) * kTok;
    const bool live = c0 < p.C && tfirst < p.T;
    const int t0 = live ? static_cast<int>(tfirst) : 0;
    const int t1 = live ? min(t0 + kTok, p.T) : 0;  // this thread's tokens

    float2 sum[K + 1][2];  // BWD: dw by distance back, then dbias
#pragma unroll
    for (int d = 0; d <= K; ++d) sum[d][0] = sum[d][1] = splat2(0.0f);

    if (live) {
        const T* u = static_cast<const T*>(p.u) + b * p.usb + c0;
        const T* go = BWD ? static_cast<const T*>(p.gout) + b * p.gsb + c0 : nullptr;
        T* out = static_cast<T*>(p.out) + int64_t(b) * p.T * p.C + c0;
        const uint8_t* seg = p.seg != nullptr ? p.seg + b * p.sgb : nullptr;
        float2 w[K][2], bs[2];  // w[d]: the tap that multiplies the input d tokens back
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            bs[i] = p.bias != nullptr ? make_float2(p.bias[c0 + 2 * i], p.bias[c0 + 2 * i + 1]) : splat2(0.0f);
#pragma unroll
            for (int d = 0; d < K; ++d)
                w[d][i] = make_float2(p.w[int64_t(c0 + 2 * i) * K + K - 1 - d], p.w[int64_t(c0 + 2 * i + 1) * K + K - 1 - d]);
        }
        float2 win[H][2], du[K][2];  // the inputs 1..K-1 tokens back; BWD: du of the token d back
#pragma unroll
        for (int d = 0; d < H; ++d) win[d][0] = win[d][1] = splat2(0.0f);
#pragma unroll
        for (int d = 0; d < K; ++d) du[d][0] = du[d][1] = splat2(0.0f);
        auto push = [&](const float2 (&x)[2]) {
#pragma unroll
            for (int d = H - 1; d >= 1; --d) win[d][0] = win[d - 1][0], win[d][1] = win[d - 1][1];
            win[0][0] = x[0], win[0][1] = x[1];
        };
        auto cut = [&]() {  // a segment starts: the inputs before it are out of reach
#pragma unroll
            for (int d = 0; d < H; ++d) win[d][0] = win[d][1] = splat2(0.0f);
        };
        auto starts = [&](int t) { return seg != nullptr && seg[int64_t(t) * p.sgt] != 0; };
        if constexpr (K > 1) {
#pragma unroll
            for (int d = K - 1; d >= 1; --d) {
                const int t = t0 - d;
                if (t < 0) continue;
                if (starts(t)) cut();
                float2 x[2];
                load4<T>(u + int64_t(t) * p.ust, x);
                push(x);
            }
        }
        int back = -1;  // BWD: tokens before t, from t0 on, in t's segment (at most K-1 matter)
        const int tend = BWD ? t1 + K - 1 : t1;
        for (int tg = t0; tg < tend; tg += kAhead) {
            float2 x[kAhead][2], g[kAhead][2];
            bool st[kAhead];
#pragma unroll
            for (int i = 0; i < kAhead; ++i) {
                const int t = tg + i;
                x[i][0] = x[i][1] = g[i][0] = g[i][1] = splat2(0.0f);
                st[i] = false;
                if (t < tend && t < p.T) {
                    load4<T>(u + int64_t(t) * p.ust, x[i]);
                    if constexpr (BWD) load4<T>(go + int64_t(t) * p.gst, g[i]);
                    st[i] = starts(t);
                }
            }
#pragma unroll
            for (int i = 0; i < kAhead; ++i) {
                const int t = tg + i;
                if (t >= tend) break;
                if (st[i]) cut();
                float2 y[2];
                if constexpr (BWD) {
                    back = st[i] ? 0 : back + 1;
#pragma unroll
                    for (int d = K - 1; d >= 1; --d) du[d][0] = du[d - 1][0], du[d][1] = du[d - 1][1];
                    du[0][0] = du[0][1] = splat2(0.0f);
                }
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float2 v = bs[e];
#pragma unroll
                    for (int d = K - 1; d >= 0; --d) v = ffma2(w[d][e], d == 0 ? x[i][e] : win[d > 0 ? d - 1 : 0][e], v);
                    float2 s, n;
                    sig_pair<T>(v, s, n);
                    if constexpr (!BWD) {
                        y[e] = fmul2(v, s);
                    } else {
                        const float2 dv = fmul2(fmul2(g[i][e], s), ffma2(v, n, splat2(1.0f)));
#pragma unroll
                        for (int d = 0; d < K; ++d)
                            if (d <= back) du[d][e] = ffma2(w[d][e], dv, du[d][e]);
                        if (t < t1) {
                            sum[K][e] = fadd2(sum[K][e], dv);
#pragma unroll
                            for (int d = 0; d < K; ++d)
                                sum[d][e] = ffma2(dv, d == 0 ? x[i][e] : win[d > 0 ? d - 1 : 0][e], sum[d][e]);
                        }
                    }
                }
                push(x[i]);
                if constexpr (!BWD) {
                    store4<T>(out + int64_t(t) * p.C, y);
                } else {
                    const int td = t - (K - 1);  // this token has met every dv it feeds
                    if (td >= t0 && td < t1) store4<T>(out + int64_t(td) * p.C, du[K - 1]);
                }
            }
        }
    }
    if constexpr (BWD) {
        __shared__ float2 s_sum[kRanges][(K + 1) * 2][32];
#pragma unroll
        for (int d = 0; d <= K; ++d)
#pragma unroll
            for (int e = 0; e < 2; ++e) s_sum[threadIdx.y][2 * d + e][threadIdx.x] = sum[d][e];
        __syncthreads();
        float* part = p.part + (int64_t(b) * p.ntb + tb) * int64_t(p.C) * (K + 1);
        for (int k = threadIdx.y; k < (K + 1) * 2; k += kRanges) {
            if (c0 >= p.C) continue;
            float2 t = splat2(0.0f);
#pragma unroll
            for (int r = 0; r < kRanges; ++r) t = fadd2(t, s_sum[r][k][threadIdx.x]);
            const int d = k / 2, ch = c0 + 2 * (k & 1), j = d < K ? K - 1 - d : K;
            part[int64_t(ch) * (K + 1) + j] = t.x;
            part[int64_t(ch + 1) * (K + 1) + j] = t.y;
        }
    }
}

int64_t token_blocks(int64_t T) { return (T + kTok * kRanges - 1) / (kTok * kRanges); }

template <typename T, bool BWD>
void launch_taps(int K, unsigned grid, const ConvTrainParams& p, cudaStream_t s) {
    const dim3 block(32, kRanges);
    switch (K) {
        case 1: conv_train_kernel<T, 1, BWD><<<grid, block, 0, s>>>(p); break;
        case 2: conv_train_kernel<T, 2, BWD><<<grid, block, 0, s>>>(p); break;
        case 3: conv_train_kernel<T, 3, BWD><<<grid, block, 0, s>>>(p); break;
        default: conv_train_kernel<T, 4, BWD><<<grid, block, 0, s>>>(p); break;
    }
}

template <bool BWD>
int conv_train(const need_conv_train_args* a, cudaStream_t s) {
    if (a == nullptr) return fail(NEED_ERR_INVALID, "args is null");
    if (!dtype_ok(a->dtype)) return fail(NEED_ERR_UNSUPPORTED, "conv: dtype %d", a->dtype);
    if (a->K < 1 || a->K > kMaxTaps) return fail(NEED_ERR_UNSUPPORTED, "K=%d taps (1..%d supported)", a->K, kMaxTaps);
    if (a->nb < 1 || a->T < 1 || a->C < 1) return fail(NEED_ERR_INVALID, "conv: sizes must be >= 1");
    if (a->C % 4 != 0) return fail(NEED_ERR_UNSUPPORTED, "conv: C=%lld must be a multiple of 4", (long long)a->C);
    if (a->T > INT32_MAX / 2 || a->C > INT32_MAX / 16) return fail(NEED_ERR_UNSUPPORTED, "conv: sizes too large");
    const uintptr_t al = 4 * dtype_bytes(a->dtype);
    auto rows_ok = [&](const void* p, int64_t sb, int64_t st) {
        return p != nullptr && reinterpret_cast<uintptr_t>(p) % al == 0 && (a->T == 1 || st % 4 == 0) &&
               (a->nb == 1 || sb % 4 == 0);
    };
    if (!rows_ok(a->u, a->u_stride_b, a->u_stride_t))
        return fail(NEED_ERR_UNSUPPORTED, "conv: u is null or its rows are not aligned to 4 elements");
    if (a->weight == nullptr) return fail(NEED_ERR_INVALID, "conv: weight is null");
    ConvTrainParams p{};
    p.u = a->u, p.usb = a->u_stride_b, p.ust = a->u_stride_t, p.w = a->weight, p.bias = a->bias;
    p.seg = a->seg_start, p.sgb = a->seg_stride_b, p.sgt = a->seg_stride_t;
    p.nb = int32_t(a->nb), p.T = int32_t(a->T), p.C = int32_t(a->C);
    p.ncg = int32_t((a->C + 127) / 128), p.ntb = int32_t(token_blocks(a->T));
    const int64_t blocks = int64_t(p.ncg) * p.ntb * a->nb;
    if (blocks > INT32_MAX) return fail(NEED_ERR_UNSUPPORTED, "conv: sizes too large");
    void* out = BWD ? a->grad_u : a->out;
    if (!rows_ok(out, 0, 0)) return fail(NEED_ERR_INVALID, "conv: the output is null or not aligned to 4 elements");
    p.out = out;
    if (BWD) {
        if (!rows_ok(a->gout, a->gout_stride_b, a->gout_stride_t))
            return fail(NEED_ERR_UNSUPPORTED, "conv: gout is null or its rows are not aligned to 4 elements");
        if (a->grad_wb == nullptr) return fail(NEED_ERR_INVALID, "conv: grad_wb is null");
        if (a->workspace == nullptr || a->workspace_bytes < need_conv_silu_train_workspace_size(a->K, a->nb, a->T, a->C))
            return fail(NEED_ERR_WORKSPACE, "conv: workspace missing or too small");
        p.gout = a->gout, p.gsb = a->gout_stride_b, p.gst = a->gout_stride_t;
        p.part = static_cast<float*>(a->workspace);
    }
    const unsigned grid = static_cast<unsigned>(blocks);
    if (a->dtype == NEED_F32) launch_taps<float, BWD>(a->K, grid, p, s);
    else if (a->dtype == NEED_BF16) launch_taps<__nv_bfloat16, BWD>(a->K, grid, p, s);
    else launch_taps<__half, BWD>(a->K, grid, p, s);
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return cuda_fail(e, "conv_train_kernel launch");
    if (BWD)
        if (int rc = column_sums(p.part, a->nb * p.ntb, a->C * (a->K + 1), a->grad_wb, s)) return rc;
    return ok();
}

}  // namespace

extern "C" {

size_t need_conv_silu_train_workspace_size(int32_t K, int64_t nb, int64_t T, int64_t C) {
    if (K < 1 || nb < 1 || T < 1 || C < 1) return 16;
    return size_t(nb) * size_t(token_blocks(T)) * size_t(C) * size_t(K + 1) * 4;
}
int need_conv_silu_train_forward(const need_conv_train_args* args, need_stream_t stream) {
    return conv_train<false>(args, stream);
}
int need_conv_silu_train_backward(const need_conv_train_args* args, need_stream_t stream) {
    return conv_train<true>(args, stream);
}

}  // extern "C"
