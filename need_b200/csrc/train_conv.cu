// train_conv.cu -- the SSD block's causal depthwise conv + SiLU with its
// gradient (need_conv_silu_train_forward, need_conv_silu_train_backward).
//
//   v_t = bias + sum_d w[K-1-d] u_{t-d}  (u_{t-d} in t's segment), y = v s(v)
//   dv = dy s(v) (1 + v s(-v));  du_t = sum_d w[K-1-d] dv_{t+d}  (t+d in t's segment)
//   dw[K-1-d] = sum over b, t of dv_t u_{t-d};  dbias = sum of dv
//
// All in fp32, rounded once on the way out.  Bound by HBM (4 B per 16-bit
// element forward, 6 B backward): a thread walks kTok tokens of 4 channels in
// groups of kGroupRows rows, the next group's loads in flight while it works on
// one; the last K-1 inputs, and backward the K-1 unfinished du, stay in
// registers, and v is computed again rather than kept.  The backward reads the
// K-1 rows behind its tokens a second time (L2) for the dv they need.  A thread's
// sums for dw and dbias are added over the block's token ranges in shared
// memory, and column_sums adds the blocks' rows in a fixed order.  Rows that are
// not aligned to 4 elements, and the channels of a last odd group, are read and
// written one by one.
#include "host_common.h"
#include "need_scan.h"
#include "scan_kernel.cuh"
#include "train_common.cuh"

using namespace need;

namespace {

constexpr int kMaxTaps = 4;
#ifndef K_CTOK
#define K_CTOK 32
#endif
#ifndef K_CMINB
#define K_CMINB 1
#endif
constexpr int kTok = K_CTOK;    // tokens per thread
constexpr int kGroupRows = 4;   // rows loaded together
constexpr int kRanges = 4;      // token ranges per block (threadIdx.y)

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
    int64_t osb, ost;
    float* part;  // [nb * ntb, C * (K + 1)]
    int32_t nb, T, C, ncg, ntb;      // channel groups (of 128) and token blocks
    int32_t uvec, gvec, ovec;        // rows aligned to 4 elements
};

// Four channels as loaded: packed, so that a row in flight costs few registers.
template <typename T>
struct Raw4 {
    typename Ops<T>::P h[2];
};
// n: how many of the four lie inside C.
template <typename T>
__device__ __forceinline__ Raw4<T> load4(const T* p, bool vec, int n) {
    Raw4<T> r;
    if (vec && n >= 4) {
        if constexpr (Ops<T>::BYTES == 4) {
            const float4 v = *reinterpret_cast<const float4*>(p);
            r.h[0] = make_float2(v.x, v.y);
            r.h[1] = make_float2(v.z, v.w);
        } else {
            const uint2 v = *reinterpret_cast<const uint2*>(p);
            r.h[0] = *reinterpret_cast<const typename Ops<T>::P*>(&v.x);
            r.h[1] = *reinterpret_cast<const typename Ops<T>::P*>(&v.y);
        }
    } else {
        float f[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) f[e] = e < n ? to_f(p[e]) : 0.0f;
        r.h[0] = Ops<T>::pack(f[0], f[1]);
        r.h[1] = Ops<T>::pack(f[2], f[3]);
    }
    return r;
}
template <typename T>
__device__ __forceinline__ void store4(T* p, bool vec, int n, const float2 (&f)[2]) {
    const typename Ops<T>::P h[2] = {Ops<T>::pack(f[0].x, f[0].y), Ops<T>::pack(f[1].x, f[1].y)};
    if (vec && n >= 4) {
        if constexpr (Ops<T>::BYTES == 4) *reinterpret_cast<float4*>(p) = *reinterpret_cast<const float4*>(h);
        else *reinterpret_cast<uint2*>(p) = *reinterpret_cast<const uint2*>(h);
    } else {
        const T* e = reinterpret_cast<const T*>(h);
        for (int i = 0; i < 4 && i < n; ++i) p[i] = e[i];
    }
}

template <typename T, int K, bool BWD, bool SEG>
__global__ void __launch_bounds__(32 * kRanges, K_CMINB) conv_train_kernel(const ConvTrainParams p) {
    constexpr int G = kGroupRows, W = K - 1;  // W: tokens a tap reaches back
    const int cg = blockIdx.x % p.ncg;
    const int rest = blockIdx.x / p.ncg;
    const int tb = rest % p.ntb, b = rest / p.ntb;
    const int c0 = cg * 128 + threadIdx.x * 4, n = p.C - c0;
    const int64_t tfirst = (int64_t(tb) * kRanges + threadIdx.y) * kTok;
    const bool live = n > 0 && tfirst < p.T;
    const int t0 = live ? static_cast<int>(tfirst) : 0;
    const int t1 = live ? min(t0 + kTok, p.T) : 0;  // this thread's tokens

    float2 sum[K + 1][2];  // BWD: dw by distance back, then dbias
#pragma unroll
    for (int d = 0; d <= K; ++d) sum[d][0] = sum[d][1] = splat2(0.0f);

    if (live) {
        const T* u = static_cast<const T*>(p.u) + b * p.usb + c0;
        const T* go = BWD ? static_cast<const T*>(p.gout) + b * p.gsb + c0 : nullptr;
        T* out = static_cast<T*>(p.out) + b * p.osb + c0;
        const uint8_t* seg = SEG ? p.seg + b * p.sgb : nullptr;
        float2 w[K][2], bs[2];  // w[d]: the tap that multiplies the input d tokens back
        auto param = [&](const float* q, int64_t stride, int e) { return e < n ? q[int64_t(c0 + e) * stride] : 0.0f; };
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            bs[i] = p.bias != nullptr ? make_float2(param(p.bias, 1, 2 * i), param(p.bias, 1, 2 * i + 1)) : splat2(0.0f);
#pragma unroll
            for (int d = 0; d < K; ++d)
                w[d][i] = make_float2(param(p.w + W - d, K, 2 * i), param(p.w + W - d, K, 2 * i + 1));
        }
        // x[W + i]: the input of the group's row i; x[0 .. W-1]: the W rows before.
        // du likewise: rows W back are finished by the group.  starts, bit W + i: row i
        // starts a segment.
        float2 x[W + G][2], du[W + G][2];
        uint32_t starts = 0;
#pragma unroll
        for (int d = 0; d < W; ++d) {
            x[d][0] = x[d][1] = du[d][0] = du[d][1] = splat2(0.0f);
            const int t = t0 - W + d;
            if (t >= 0) {
                const Raw4<T> r = load4<T>(u + int64_t(t) * p.ust, p.uvec != 0, n);
                x[d][0] = widen(r.h[0]);
                x[d][1] = widen(r.h[1]);
                if (SEG && seg[int64_t(t) * p.sgt] != 0) starts |= 1u << d;
            }
        }
        Raw4<T> nu[G], ng[G];  // the next group, in flight
        uint32_t nst = 0;
        auto fetch = [&](int tg) {
            nst = 0;
#pragma unroll
            for (int i = 0; i < G; ++i) {
                const int t = tg + i;
                const bool in = t < p.T && t < (BWD ? t1 + W : t1);
                nu[i].h[0] = nu[i].h[1] = Ops<T>::zero();
                if (BWD) ng[i].h[0] = ng[i].h[1] = Ops<T>::zero();
                if (in) {
                    nu[i] = load4<T>(u + int64_t(t) * p.ust, p.uvec != 0, n);
                    if constexpr (BWD) ng[i] = load4<T>(go + int64_t(t) * p.gst, p.gvec != 0, n);
                    if (SEG && seg[int64_t(t) * p.sgt] != 0) nst |= 1u << (W + i);
                }
            }
        };
        fetch(t0);
        const int tend = BWD ? t1 + W : t1;
        for (int tg = t0; tg < tend; tg += G) {
            Raw4<T> g[G];
#pragma unroll
            for (int i = 0; i < G; ++i) {
                x[W + i][0] = widen(nu[i].h[0]);
                x[W + i][1] = widen(nu[i].h[1]);
                if (BWD) g[i] = ng[i];
                du[W + i][0] = du[W + i][1] = splat2(0.0f);
            }
            starts |= nst;
            if (tg + G < tend) fetch(tg + G);
#pragma unroll
            for (int i = 0; i < G; ++i) {
                const int t = tg + i;
                // the input d back is in reach when none of the rows after it, up to t, starts a segment
                auto reach = [&](int d) { return !SEG || ((starts >> (W + i - d + 1)) & ((1u << d) - 1u)) == 0u; };
                float2 y[2];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float2 v = bs[e];
#pragma unroll
                    for (int d = W; d >= 0; --d)
                        if (reach(d)) v = ffma2(w[d][e], x[W + i - d][e], v);
                    float2 s, m;
                    sig_pair<T>(v, s, m);
                    if constexpr (!BWD) {
                        y[e] = fmul2(v, s);
                    } else {
                        const float2 dv = fmul2(fmul2(widen(g[i].h[e]), s), ffma2(v, m, splat2(1.0f)));
#pragma unroll
                        for (int d = 0; d < K; ++d)
                            if (reach(d)) du[W + i - d][e] = ffma2(w[d][e], dv, du[W + i - d][e]);
                        if (t < t1) {
                            sum[K][e] = fadd2(sum[K][e], dv);
#pragma unroll
                            for (int d = 0; d < K; ++d)
                                if (reach(d)) sum[d][e] = ffma2(dv, x[W + i - d][e], sum[d][e]);
                        }
                    }
                }
                if constexpr (!BWD)
                    if (t < t1) store4<T>(out + int64_t(t) * p.ost, p.ovec != 0, n, y);
            }
            if constexpr (BWD) {
#pragma unroll
                for (int i = 0; i < G; ++i) {  // these rows have met every dv they feed
                    const int t = tg - W + i;
                    if (t >= t0 && t < t1) store4<T>(out + int64_t(t) * p.ost, p.ovec != 0, n, du[i]);
                }
            }
#pragma unroll
            for (int d = 0; d < W; ++d)
#pragma unroll
                for (int e = 0; e < 2; ++e) x[d][e] = x[G + d][e], du[d][e] = du[G + d][e];
            starts >>= G;
        }
        if constexpr (BWD && W > 0) {  // rows the last group left behind
#pragma unroll
            for (int d = 0; d < W; ++d) {
                const int t = t0 + (tend - t0 + G - 1) / G * G - W + d;
                if (t >= t0 && t < t1) store4<T>(out + int64_t(t) * p.ost, p.ovec != 0, n, du[d]);
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
            float2 t = splat2(0.0f);
#pragma unroll
            for (int r = 0; r < kRanges; ++r) t = fadd2(t, s_sum[r][k][threadIdx.x]);
            const int d = k / 2, ch = c0 + 2 * (k & 1), j = d < K ? W - d : K;
            if (ch < p.C) part[int64_t(ch) * (K + 1) + j] = t.x;
            if (ch + 1 < p.C) part[int64_t(ch + 1) * (K + 1) + j] = t.y;
        }
    }
}

int64_t token_blocks(int64_t T) { return (T + kTok * kRanges - 1) / (kTok * kRanges); }

template <typename T, bool BWD, bool SEG>
void launch_taps(int K, unsigned grid, const ConvTrainParams& p, cudaStream_t s) {
    const dim3 block(32, kRanges);
    switch (K) {
        case 1: conv_train_kernel<T, 1, BWD, SEG><<<grid, block, 0, s>>>(p); break;
        case 2: conv_train_kernel<T, 2, BWD, SEG><<<grid, block, 0, s>>>(p); break;
        case 3: conv_train_kernel<T, 3, BWD, SEG><<<grid, block, 0, s>>>(p); break;
        default: conv_train_kernel<T, 4, BWD, SEG><<<grid, block, 0, s>>>(p); break;
    }
}

template <bool BWD>
int conv_train(const need_conv_train_args* a, cudaStream_t s) {
    if (a == nullptr) return fail(NEED_ERR_INVALID, "args is null");
    if (!dtype_ok(a->dtype)) return fail(NEED_ERR_UNSUPPORTED, "conv: dtype %d", a->dtype);
    if (a->K < 1 || a->K > kMaxTaps) return fail(NEED_ERR_UNSUPPORTED, "K=%d taps (1..%d supported)", a->K, kMaxTaps);
    if (a->nb < 1 || a->T < 1 || a->C < 1) return fail(NEED_ERR_INVALID, "conv: sizes must be >= 1");
    if (a->nb > INT32_MAX || a->T > INT32_MAX / 2 || a->C > INT32_MAX / 16)
        return fail(NEED_ERR_UNSUPPORTED, "conv: sizes too large");
    if (a->u == nullptr) return fail(NEED_ERR_INVALID, "conv: u is null");
    if (a->weight == nullptr) return fail(NEED_ERR_INVALID, "conv: weight is null");
    const uintptr_t al = 4 * dtype_bytes(a->dtype);
    auto vec = [&](const void* q, int64_t sb, int64_t st) {
        return reinterpret_cast<uintptr_t>(q) % al == 0 && (a->T == 1 || st % 4 == 0) && (a->nb == 1 || sb % 4 == 0);
    };
    ConvTrainParams p{};
    p.u = a->u, p.usb = a->u_stride_b, p.ust = a->u_stride_t, p.w = a->weight, p.bias = a->bias;
    p.seg = a->seg_start, p.sgb = a->seg_stride_b, p.sgt = a->seg_stride_t;
    p.nb = int32_t(a->nb), p.T = int32_t(a->T), p.C = int32_t(a->C);
    p.ncg = int32_t((a->C + 127) / 128), p.ntb = int32_t(token_blocks(a->T));
    const int64_t blocks = int64_t(p.ncg) * p.ntb * a->nb;
    if (int64_t(p.ncg) * p.ntb > INT32_MAX || blocks > INT32_MAX) return fail(NEED_ERR_UNSUPPORTED, "conv: sizes too large");
    p.out = BWD ? a->grad_u : a->out;
    if (p.out == nullptr) return fail(NEED_ERR_INVALID, "conv: the output is null");
    p.osb = a->out_stride_b, p.ost = a->out_stride_t;
    if (a->T > 1 && p.ost < a->C) return fail(NEED_ERR_INVALID, "conv: the output's rows overlap");
    p.uvec = vec(p.u, p.usb, p.ust), p.ovec = vec(p.out, p.osb, p.ost);
    if (BWD) {
        if (a->gout == nullptr) return fail(NEED_ERR_INVALID, "conv: gout is null");
        if (a->grad_wb == nullptr) return fail(NEED_ERR_INVALID, "conv: grad_wb is null");
        if (a->workspace == nullptr || a->workspace_bytes < need_conv_silu_train_workspace_size(a->K, a->nb, a->T, a->C))
            return fail(NEED_ERR_WORKSPACE, "conv: workspace missing or too small");
        p.gout = a->gout, p.gsb = a->gout_stride_b, p.gst = a->gout_stride_t;
        p.gvec = vec(p.gout, p.gsb, p.gst);
        p.part = static_cast<float*>(a->workspace);
    }
    const unsigned grid = static_cast<unsigned>(blocks);
    auto go = [&](auto tag) {
        using T = decltype(tag);
        if (p.seg != nullptr) launch_taps<T, BWD, true>(a->K, grid, p, s);
        else launch_taps<T, BWD, false>(a->K, grid, p, s);
    };
    if (a->dtype == NEED_F32) go(float{});
    else if (a->dtype == NEED_BF16) go(__nv_bfloat16{});
    else go(__half{});
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
