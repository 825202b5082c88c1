// train_conv.cu -- the SSD block's causal depthwise conv + SiLU with its
// gradient (need_conv_silu_train_forward, need_conv_silu_train_backward).
//
//   v_t = bias + sum_d w[K-1-d] u_{t-d}  (u_{t-d} in t's segment), y = v s(v)
//   dv = dy s(v) (1 + v s(-v));  du_t = sum_d w[K-1-d] dv_{t+d}  (t+d in t's segment)
//   dw[K-1-d] = sum over b, t of dv_t u_{t-d};  dbias = sum of dv
//
// All in fp32, rounded once on the way out.  A thread walks its tokens of 4
// channels (backward 2) in groups of kGroupRows rows.  The next groups are on their
// way into shared memory meanwhile, copied asynchronously to places that only this
// thread reads, so that rows in flight cost no registers.  The last K-1 inputs, and
// backward the K-1 unfinished du, stay in registers, and v is computed again rather
// than kept.  The backward reads the K-1 rows behind its tokens a second time (L2)
// for the dv they need.  A thread's sums for dw and dbias are added over the block's
// token ranges in shared memory, and column_sums adds the blocks' rows in a fixed
// order.  Rows that are not aligned to a thread's channels, and a last partial group, are
// copied a 4-byte word at a time, 16-bit ones that lie between words loaded one by one
// (8x2048 bf16: C = 832 39 us the pass, 830 44, 831 136).
//
// What bounds it (B200, bf16, K = 3): 4 B move per element forward, 6 B backward;
// 8x2048x832 12 us (4.5 TB/s) and 25 us (3.3 TB/s), 16x4096x1024 146 us the pass (4.6
// TB/s).  Nothing is full backward (58 % of the issue slots, 25 % of the warps active): a
// thread's walk over its rows, in one wave and a fifth.  With the next group in registers
// in place of shared memory, one group ahead and 32 tokens, the passes took 45 and 180 us.
#include <string.h>

#include <type_traits>

#include "host_common.h"
#include "need_scan.h"
#include "scan_kernel.cuh"
#include "train_common.cuh"

using namespace need;

namespace {

constexpr int kMaxTaps = 4;
constexpr int kGroupRows = 4;   // rows loaded together
constexpr int kRanges = 4;      // token ranges per block (threadIdx.y)
constexpr int kStages = 3;      // groups in shared memory: one worked on, two on their way
constexpr int kBlocks = 5;      // per SM (96 registers); 6 spill and measured the same
// Channel pairs per thread.  The backward keeps du, the sums and a second stream
// besides: two pairs took 182 registers, 2 blocks per SM and 44 us (29 us with one) at
// 8x2048x832 bf16, K = 3.
template <bool BWD>
constexpr int kPairs = BWD ? 1 : 2;

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
    int32_t tok;   // tokens per thread
    int32_t nb, T, C, ncg, ntb;      // channel groups (of 32 threads) and token blocks
    int32_t uvec, gvec, ovec;        // rows aligned to a thread's channels
    int32_t words;                   // u's and gout's to 4 bytes
};

// 2 NP channels as loaded: packed, so that a row in flight costs few registers.
template <typename T, int NP>
struct Raw {
    typename Ops<T>::P h[NP];
};
// n: how many of the channels lie inside C.
template <typename T, int NP>
__device__ __forceinline__ Raw<T, NP> load_row(const T* p, bool vec, int n) {
    using V = typename std::conditional<sizeof(Raw<T, NP>) == 16, uint4,
                                        typename std::conditional<sizeof(Raw<T, NP>) == 8, uint2, uint32_t>::type>::type;
    Raw<T, NP> r;
    if (vec && n >= 2 * NP) {
        const V v = *reinterpret_cast<const V*>(p);
        memcpy(&r, &v, sizeof(v));
    } else {
#pragma unroll
        for (int e = 0; e < NP; ++e)
            r.h[e] = Ops<T>::pack(2 * e < n ? to_f(p[2 * e]) : 0.0f, 2 * e + 1 < n ? to_f(p[2 * e + 1]) : 0.0f);
    }
    return r;
}
// BYTES of a row to this thread's place in shared memory, asynchronously; `in` false: zeros.
template <int BYTES>
__device__ __forceinline__ void copy_async(void* dst, const void* src, bool in) {
    const uint32_t d = static_cast<uint32_t>(__cvta_generic_to_shared(dst));
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(d), "l"(src), "n"(BYTES), "r"(in ? BYTES : 0)
                 : "memory");
}
template <typename T, int NP>
__device__ __forceinline__ void store_row(T* p, bool vec, int n, const float2 (&f)[NP]) {
    using V = typename std::conditional<sizeof(Raw<T, NP>) == 16, uint4,
                                        typename std::conditional<sizeof(Raw<T, NP>) == 8, uint2, uint32_t>::type>::type;
    Raw<T, NP> r;
#pragma unroll
    for (int e = 0; e < NP; ++e) r.h[e] = Ops<T>::pack(f[e].x, f[e].y);
    if (vec && n >= 2 * NP) {
        V v;
        memcpy(&v, &r, sizeof(v));
        *reinterpret_cast<V*>(p) = v;
    } else {
        const T* e = reinterpret_cast<const T*>(&r);
        for (int i = 0; i < 2 * NP && i < n; ++i) p[i] = e[i];
    }
}

template <typename T, int K, bool BWD, bool SEG>
__global__ void __launch_bounds__(32 * kRanges, kBlocks) conv_train_kernel(const ConvTrainParams p) {
    constexpr int G = kGroupRows, W = K - 1;  // W: tokens a tap reaches back
    constexpr int NP = kPairs<BWD>, NC = 2 * NP;
    const int cg = blockIdx.x % p.ncg;
    const int rest = blockIdx.x / p.ncg;
    const int tb = rest % p.ntb, b = rest / p.ntb;
    const int c0 = (cg * 32 + threadIdx.x) * NC, n = p.C - c0;
    const int64_t tfirst = (int64_t(tb) * kRanges + threadIdx.y) * p.tok;
    const bool live = n > 0 && tfirst < p.T;
    const int t0 = live ? static_cast<int>(tfirst) : 0;
    const int t1 = live ? min(t0 + p.tok, p.T) : 0;  // this thread's tokens

    // a ring of kStages groups, each thread's own places: [stage][row][thread]
    using Place = Raw<T, NP>;
    __shared__ __align__(16) Place s_u[kStages * G][32 * kRanges];
    __shared__ __align__(16) Place s_g[BWD ? kStages * G : 1][32 * kRanges];
    const int tid = threadIdx.y * 32 + threadIdx.x;

    float2 sum[K + 1][NP];  // BWD: dw by distance back, then dbias
#pragma unroll
    for (int d = 0; d <= K; ++d)
#pragma unroll
        for (int e = 0; e < NP; ++e) sum[d][e] = splat2(0.0f);

    if (live) {
        const T* u = static_cast<const T*>(p.u) + b * p.usb + c0;
        const T* go = BWD ? static_cast<const T*>(p.gout) + b * p.gsb + c0 : nullptr;
        T* out = static_cast<T*>(p.out) + b * p.osb + c0;
        const uint8_t* seg = SEG ? p.seg + b * p.sgb : nullptr;
        const int tend = BWD ? t1 + W : t1, tin = min(tend, p.T);
        const bool vec = p.uvec != 0 && p.ovec != 0 && (!BWD || p.gvec != 0) && n >= NC;
        constexpr int PW = 4 / sizeof(T);  // elements of a word
        const bool words = p.words != 0 && n % PW == 0;
        const T* fu = u + int64_t(t0) * p.ust;  // the first row of the group fetched next
        const T* fg = BWD ? go + int64_t(t0) * p.gst : nullptr;
        int ft = t0, fs = 0;  // its token and its stage's first place
        auto fetch = [&] {
            if (vec && ft + G <= tin) {
#pragma unroll
                for (int i = 0; i < G; ++i) {
                    copy_async<sizeof(Place)>(&s_u[fs + i][tid], fu + i * p.ust, true);
                    if constexpr (BWD) copy_async<sizeof(Place)>(&s_g[fs + i][tid], fg + i * p.gst, true);
                }
            } else if (words && ft < tend) {
#pragma unroll
                for (int i = 0; i < G; ++i) {
                    const bool ok = ft + i < tin;
#pragma unroll
                    for (int w = 0; w < NC; w += PW) {
                        const bool in = ok && w < n;
                        copy_async<4>(reinterpret_cast<T*>(&s_u[fs + i][tid]) + w, in ? fu + i * p.ust + w : u, in);
                        if constexpr (BWD)
                            copy_async<4>(reinterpret_cast<T*>(&s_g[fs + i][tid]) + w, in ? fg + i * p.gst + w : go, in);
                    }
                }
            } else if (ft < tend) {
                Place a[G], b[G];  // loaded together
#pragma unroll
                for (int i = 0; i < G; ++i) {
                    a[i] = load_row<T, NP>(fu + i * p.ust, false, ft + i < tin ? n : 0);
                    if constexpr (BWD) b[i] = load_row<T, NP>(fg + i * p.gst, false, ft + i < tin ? n : 0);
                }
#pragma unroll
                for (int i = 0; i < G; ++i) {
                    s_u[fs + i][tid] = a[i];
                    if constexpr (BWD) s_g[fs + i][tid] = b[i];
                }
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
            fu += G * p.ust;
            if (BWD) fg += G * p.gst;
            ft += G;
            fs = fs == (kStages - 1) * G ? 0 : fs + G;
        };
#pragma unroll
        for (int k = 0; k < kStages - 1; ++k) fetch();
        float2 w[K][NP], bs[NP];  // w[d]: the tap that multiplies the input d tokens back
        auto param = [&](const float* q, int64_t stride, int e) { return e < n ? q[int64_t(c0 + e) * stride] : 0.0f; };
#pragma unroll
        for (int i = 0; i < NP; ++i) {
            bs[i] = p.bias != nullptr ? make_float2(param(p.bias, 1, 2 * i), param(p.bias, 1, 2 * i + 1)) : splat2(0.0f);
#pragma unroll
            for (int d = 0; d < K; ++d)
                w[d][i] = make_float2(param(p.w + W - d, K, 2 * i), param(p.w + W - d, K, 2 * i + 1));
        }
        // x[W + i]: the input of the group's row i; x[0 .. W-1]: the W rows before.
        // du likewise: rows W back are finished by the group.  starts, bit W + i: row i
        // starts a segment.
        float2 x[W + G][NP], du[W + G][NP];
        uint32_t starts = 0;
#pragma unroll
        for (int d = 0; d < W; ++d) {
#pragma unroll
            for (int e = 0; e < NP; ++e) x[d][e] = du[d][e] = splat2(0.0f);
            const int t = t0 - W + d;
            if (t >= 0) {
                const Raw<T, NP> r = load_row<T, NP>(u + int64_t(t) * p.ust, p.uvec != 0, n);
#pragma unroll
                for (int e = 0; e < NP; ++e) x[d][e] = widen(r.h[e]);
                if (SEG && seg[int64_t(t) * p.sgt] != 0) starts |= 1u << d;
            }
        }
        uint32_t nst = 0;  // the next group's segment starts
        auto marks = [&](int tg) {
            nst = 0;
            if constexpr (SEG) {
#pragma unroll
                for (int i = 0; i < G; ++i)
                    if (tg + i < tin && seg[int64_t(tg + i) * p.sgt] != 0) nst |= 1u << (W + i);
            }
        };
        int rs = 0;  // the first place of the group worked on
        T* orow = out + int64_t(t0 - (BWD ? W : 0)) * p.ost;  // the row the group finishes first
        auto group = [&](int tg, auto all) {
            constexpr bool ALL = decltype(all)::value;  // all rows are this thread's, and so are those it finishes
            asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 2) : "memory");
            Place g[G];
#pragma unroll
            for (int i = 0; i < G; ++i) {
                const Place r = s_u[rs + i][tid];
#pragma unroll
                for (int e = 0; e < NP; ++e) x[W + i][e] = widen(r.h[e]), du[W + i][e] = splat2(0.0f);
                if (BWD) g[i] = s_g[rs + i][tid];
            }
            rs = rs == (kStages - 1) * G ? 0 : rs + G;
            starts |= nst;
            marks(tg + G);
            fetch();  // into the places of the group before this one
#pragma unroll
            for (int i = 0; i < G; ++i) {
                // the input d back is in reach when none of the rows after it, up to this one, starts a segment
                auto reach = [&](int d) { return !SEG || ((starts >> (W + i - d + 1)) & ((1u << d) - 1u)) == 0u; };
                float2 y[NP];
#pragma unroll
                for (int e = 0; e < NP; ++e) {
                    float2 v = bs[e];
#pragma unroll
                    for (int d = W; d >= 0; --d)
                        if (reach(d)) v = ffma2(w[d][e], x[W + i - d][e], v);
                    float2 s, m;
                    sig_pair<T>(v, s, m);
                    if constexpr (!BWD) {
                        y[e] = fmul2(v, s);
                    } else {
                        float2 dv = fmul2(fmul2(widen(g[i].h[e]), s), ffma2(v, m, splat2(1.0f)));
                        // behind the sequence gout is 0, but v may be past fp32 where none of its rows is
                        if (!ALL && tg + i >= tin) dv = splat2(0.0f);
#pragma unroll
                        for (int d = 0; d < K; ++d)
                            if (reach(d)) du[W + i - d][e] = ffma2(w[d][e], dv, du[W + i - d][e]);
                        if (ALL || tg + i < t1) {
                            sum[K][e] = fadd2(sum[K][e], dv);
#pragma unroll
                            for (int d = 0; d < K; ++d)
                                if (reach(d)) sum[d][e] = ffma2(dv, x[W + i - d][e], sum[d][e]);
                        }
                    }
                }
                if constexpr (!BWD)
                    if (ALL || tg + i < t1)
                        store_row<T, NP>(orow + i * p.ost, ALL || p.ovec != 0, ALL ? NC : n, y);
            }
            if constexpr (BWD) {
#pragma unroll
                for (int i = 0; i < G; ++i)  // these rows have met every dv they feed
                    if (ALL || (tg - W + i >= t0 && tg - W + i < t1))
                        store_row<T, NP>(orow + i * p.ost, ALL || p.ovec != 0, ALL ? NC : n, du[i]);
            }
            orow += G * p.ost;
#pragma unroll
            for (int d = 0; d < W; ++d)
#pragma unroll
                for (int e = 0; e < NP; ++e) x[d][e] = x[G + d][e], du[d][e] = du[G + d][e];
            starts >>= G;
        };

        marks(t0);
        for (int tg = t0; tg < tend; tg += G) {
            if (vec && tg + G <= t1 && (!BWD || tg - W >= t0)) group(tg, std::true_type{});
            else group(tg, std::false_type{});
        }
        if constexpr (BWD && W > 0) {  // rows the last group left behind
#pragma unroll
            for (int d = 0; d < W; ++d) {
                const int t = t0 + (tend - t0 + G - 1) / G * G - W + d;
                if (t >= t0 && t < t1) store_row<T, NP>(out + int64_t(t) * p.ost, p.ovec != 0, n, du[d]);
            }
        }
    }
    if constexpr (BWD) {
        __shared__ float2 s_sum[kRanges][(K + 1) * NP][32];
#pragma unroll
        for (int d = 0; d <= K; ++d)
#pragma unroll
            for (int e = 0; e < NP; ++e) s_sum[threadIdx.y][NP * d + e][threadIdx.x] = sum[d][e];
        __syncthreads();
        float* part = p.part + (int64_t(b) * p.ntb + tb) * int64_t(p.C) * (K + 1);
        for (int k = threadIdx.y; k < (K + 1) * NP; k += kRanges) {
            float2 t = splat2(0.0f);
#pragma unroll
            for (int r = 0; r < kRanges; ++r) t = fadd2(t, s_sum[r][k][threadIdx.x]);
            const int d = k / NP, ch = c0 + 2 * (k % NP), j = d < K ? W - d : K;
            if (ch < p.C) part[int64_t(ch) * (K + 1) + j] = t.x;
            if (ch + 1 < p.C) part[int64_t(ch + 1) * (K + 1) + j] = t.y;
        }
    }
}

// Tokens per thread: 64 where that leaves enough threads, down to 16 where a
// thread's walk is what the call waits for (B200 device us of a bf16 pass, K = 3, at
// 16 / 32 / 64 / 128 tokens both ways: 16x4096x1024 202 / 161 / 146 / 147, 8x2048x832
// 46.9 / 41.7 / 40.8 / -, 4x1024x832 18.5 / 17.2 / 20.0 / 27.7, 1x1024x2048 13.5 / 14.1 /
// 17.8 / 27.3).
int tokens(bool bwd, int64_t nb, int64_t T, int64_t C) {
    const int64_t nc = 2 * (bwd ? kPairs<true> : kPairs<false>);
    int t = 64;
    while (t > 16 && nb * ((T + t - 1) / t) * ((C + nc - 1) / nc) < 1480 * t) t /= 2;
    return t;
}
int64_t token_blocks(bool bwd, int64_t nb, int64_t T, int64_t C) {
    const int64_t t = int64_t(tokens(bwd, nb, T, C)) * kRanges;
    return (T + t - 1) / t;
}

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
    constexpr int NC = 2 * kPairs<BWD>;
    const uintptr_t al = NC * dtype_bytes(a->dtype);
    auto vec = [&](const void* q, int64_t sb, int64_t st) {
        return reinterpret_cast<uintptr_t>(q) % al == 0 && (a->T == 1 || st % NC == 0) && (a->nb == 1 || sb % NC == 0);
    };
    ConvTrainParams p{};
    p.u = a->u, p.usb = a->u_stride_b, p.ust = a->u_stride_t, p.w = a->weight, p.bias = a->bias;
    p.seg = a->seg_start, p.sgb = a->seg_stride_b, p.sgt = a->seg_stride_t;
    p.nb = int32_t(a->nb), p.T = int32_t(a->T), p.C = int32_t(a->C);
    p.ncg = int32_t((a->C + 64 * kPairs<BWD> - 1) / (64 * kPairs<BWD>)), p.ntb = int32_t(token_blocks(BWD, a->nb, a->T, a->C));
    p.tok = tokens(BWD, a->nb, a->T, a->C);
    const int64_t blocks = int64_t(p.ncg) * p.ntb * a->nb;
    if (int64_t(p.ncg) * p.ntb > INT32_MAX || blocks > INT32_MAX) return fail(NEED_ERR_UNSUPPORTED, "conv: sizes too large");
    p.out = BWD ? a->grad_u : a->out;
    if (p.out == nullptr) return fail(NEED_ERR_INVALID, "conv: the output is null");
    p.osb = a->out_stride_b, p.ost = a->out_stride_t;
    if (a->T > 1 && p.ost < a->C) return fail(NEED_ERR_INVALID, "conv: the output's rows overlap");
    auto words = [&](const void* q, int64_t sb, int64_t st) {
        const int64_t n = 4 / dtype_bytes(a->dtype);
        return reinterpret_cast<uintptr_t>(q) % 4 == 0 && (a->T == 1 || st % n == 0) && (a->nb == 1 || sb % n == 0);
    };
    p.words = words(p.u, p.usb, p.ust) && (!BWD || words(a->gout, a->gout_stride_b, a->gout_stride_t));
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
    return size_t(nb) * size_t(token_blocks(true, nb, T, C)) * size_t(C) * size_t(K + 1) * 4;
}
int need_conv_silu_train_forward(const need_conv_train_args* args, need_stream_t stream) {
    return conv_train<false>(args, stream);
}
int need_conv_silu_train_backward(const need_conv_train_args* args, need_stream_t stream) {
    return conv_train<true>(args, stream);
}

}  // extern "C"
