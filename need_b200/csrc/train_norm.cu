// train_norm.cu -- RMSNorm with its gradient (need_rms_norm_train_forward,
// need_rms_norm_train_backward), the block's out_norm under training, and the
// fixed-order column sum the training kernels end with.
//
//   r = 1 / sqrt(sum(x^2) / C + eps), n = x r
//   y = n w;  g = w dy:  dx = r (g - n sum(g n) / C),  dw = sum over rows of dy n
//
// Bound by HBM: 4 B per 16-bit element forward, 6 B backward (5 and 5 with x
// kept in 8 bits).  A row is read once into the registers of 1 to 16 warps --
// the fewest that leave a lane at most 4 16-byte pieces -- and the two sums of
// the backward are reduced together.  The backward's blocks stride over the
// rows, so that a lane's channels stay the same and their share of dw stays in
// its registers; each block ends with one row of partial sums, and
// column_sums adds those rows in a fixed order.
#include <cuda_fp8.h>

#include <algorithm>

#include "host_common.h"
#include "need_scan.h"
#include "scan_kernel.cuh"
#include "train_common.cuh"

using namespace need;

namespace {

constexpr int kPieces = 4;      // 16-byte pieces per lane
constexpr int kMaxWarps = 16;   // warps per row
constexpr int kGroup = 64;      // channels per 8-bit scale

struct NormTrainParams {
    const void* x;
    int64_t xs;
    const void* gout;
    int64_t gs;
    const float* w;
    void* out;  // y, or dx
    float* rstd;
    uint8_t* q;
    uint8_t* qs;
    float* part;  // [gridDim.x, C]
    int64_t rows;
    int32_t C, ngroups, wpr;  // warps per row
    float inv_c, eps;
};

// Sums a and b over the warps of a row (all of them call it).
__device__ __forceinline__ void row_sums(float& a, float& b, int wpr, float2* s_red) {
#pragma unroll
    for (int m = 16; m >= 1; m >>= 1) {
        a += __shfl_xor_sync(0xffffffffu, a, m);
        b += __shfl_xor_sync(0xffffffffu, b, m);
    }
    if (wpr > 1) {
        const int warp = threadIdx.x >> 5;
        __syncthreads();  // the previous row's sums have been read
        if ((threadIdx.x & 31) == 0) s_red[warp] = make_float2(a, b);
        __syncthreads();
        const int w0 = warp / wpr * wpr;
        a = b = 0.0f;
        for (int w = 0; w < wpr; ++w) {
            a += s_red[w0 + w].x;
            b += s_red[w0 + w].y;
        }
    }
}

template <typename T>
struct Piece {  // a 16-byte piece of a row
    static constexpr int N = 16 / Ops<T>::BYTES;
    static __device__ __forceinline__ void load(const T* p, float2 (&f)[N / 2]) {
        const uint4 u = *reinterpret_cast<const uint4*>(p);
        const typename Ops<T>::P* h = reinterpret_cast<const typename Ops<T>::P*>(&u);
#pragma unroll
        for (int e = 0; e < N / 2; ++e) f[e] = widen(h[e]);
    }
    static __device__ __forceinline__ void store(T* p, const float2 (&f)[N / 2]) {
        uint4 u;
        typename Ops<T>::P* h = reinterpret_cast<typename Ops<T>::P*>(&u);
#pragma unroll
        for (int e = 0; e < N / 2; ++e) h[e] = Ops<T>::pack(f[e].x, f[e].y);
        *reinterpret_cast<uint4*>(p) = u;
    }
    static __device__ __forceinline__ void load_w(const float* w, float2 (&f)[N / 2]) {
#pragma unroll
        for (int e = 0; e < N / 4; ++e) {
            const float4 v = __ldg(reinterpret_cast<const float4*>(w) + e);
            f[2 * e] = make_float2(v.x, v.y);
            f[2 * e + 1] = make_float2(v.z, v.w);
        }
    }
};

// blockDim = 32 * wpr * (rows per block); a row is handled by wpr warps, lane l
// of its warp w holding pieces (w * 32 + l) + k * 32 * wpr.
template <typename T, bool CK, int NP>
__global__ void __launch_bounds__(512) norm_train_fwd(const NormTrainParams p) {
    using Pc = Piece<T>;
    constexpr int N = Pc::N;
    __shared__ float2 s_red[kMaxWarps];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rpb = (blockDim.x >> 5) / p.wpr;
    const int64_t row = int64_t(blockIdx.x) * rpb + warp / p.wpr;
    const bool live = row < p.rows;
    const int l0 = (warp % p.wpr) * 32 + lane, step = 32 * p.wpr, nvec = p.C / N;
    const T* x = static_cast<const T*>(p.x) + (live ? row : 0) * p.xs;
    float2 f[NP][N / 2];
    float ss = 0.0f, none = 0.0f;
#pragma unroll
    for (int k = 0; k < NP; ++k) {
        const int v = l0 + k * step;
#pragma unroll
        for (int e = 0; e < N / 2; ++e) f[k][e] = splat2(0.0f);
        if (live && v < nvec) Pc::load(x + v * N, f[k]);
    }
#pragma unroll
    for (int k = 0; k < NP; ++k)
#pragma unroll
        for (int e = 0; e < N / 2; ++e) ss = fmaf(f[k][e].x, f[k][e].x, fmaf(f[k][e].y, f[k][e].y, ss));
    row_sums(ss, none, p.wpr, s_red);
    const float r = 1.0f / sqrtf(fmaf(ss, p.inv_c, p.eps));
    if (live && l0 == 0) p.rstd[row] = r;
    T* out = static_cast<T*>(p.out) + row * p.C;
#pragma unroll
    for (int k = 0; k < NP; ++k) {
        const int v = l0 + k * step;
        const bool in = live && v < nvec;
        if constexpr (CK) {
            // 64 channels lie in 64 / N neighbouring lanes
            uint32_t top = 0;
#pragma unroll
            for (int e = 0; e < N / 2; ++e)
                top = max(top, max(__float_as_uint(f[k][e].x) & 0x7fffffffu, __float_as_uint(f[k][e].y) & 0x7fffffffu));
#pragma unroll
            for (int m = kGroup / N / 2; m >= 1; m >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, m));
            if (in) {
                const uint32_t sc = e4m3_scale_byte(top);
                uint16_t q[N / 2];
#pragma unroll
                for (int e = 0; e < N / 2; ++e) q[e] = e4m3_pair(f[k][e], sc);
                uint8_t* dst = p.q + row * p.C + int64_t(v) * N;
                if constexpr (N == 8)
                    *reinterpret_cast<uint2*>(dst) = make_uint2(q[0] | uint32_t(q[1]) << 16, q[2] | uint32_t(q[3]) << 16);
                else
                    *reinterpret_cast<uint32_t*>(dst) = q[0] | uint32_t(q[1]) << 16;
                if (v % (kGroup / N) == 0) p.qs[row * p.ngroups + v * N / kGroup] = static_cast<uint8_t>(sc);
            }
        }
        if (in) {
            float2 w[N / 2], o[N / 2];
            Pc::load_w(p.w + v * N, w);
#pragma unroll
            for (int e = 0; e < N / 2; ++e) o[e] = fmul2(fmul2(f[k][e], splat2(r)), w[e]);
            Pc::store(out + v * N, o);
        }
    }
}

template <typename T, bool CK, int NP>
__global__ void __launch_bounds__(512) norm_train_bwd(const NormTrainParams p) {
    using Pc = Piece<T>;
    constexpr int N = Pc::N;
    __shared__ float2 s_red[kMaxWarps];
    extern __shared__ float s_dw[];  // [C]
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rpb = (blockDim.x >> 5) / p.wpr, sub = warp / p.wpr;
    const int l0 = (warp % p.wpr) * 32 + lane, step = 32 * p.wpr, nvec = p.C / N;
    float2 dw[NP][N / 2];
#pragma unroll
    for (int k = 0; k < NP; ++k)
#pragma unroll
        for (int e = 0; e < N / 2; ++e) dw[k][e] = splat2(0.0f);
    for (int64_t base = int64_t(blockIdx.x) * rpb; base < p.rows; base += int64_t(gridDim.x) * rpb) {
        const int64_t row = base + sub;
        const bool live = row < p.rows;
        const int64_t rr = live ? row : 0;
        const T* go = static_cast<const T*>(p.gout) + rr * p.gs;
        float2 x[NP][N / 2], g[NP][N / 2];
#pragma unroll
        for (int k = 0; k < NP; ++k) {
            const int v = l0 + k * step;
#pragma unroll
            for (int e = 0; e < N / 2; ++e) x[k][e] = g[k][e] = splat2(0.0f);
            if (live && v < nvec) {
                Pc::load(go + v * N, g[k]);
                if constexpr (CK) {
                    const uint8_t* src = p.q + rr * p.C + int64_t(v) * N;
                    const float sc = e4m3_scale(p.qs[rr * p.ngroups + v * N / kGroup]);
                    uint32_t q[2] = {0, 0};
                    if constexpr (N == 8) {
                        const uint2 u = *reinterpret_cast<const uint2*>(src);
                        q[0] = u.x, q[1] = u.y;
                    } else {
                        q[0] = *reinterpret_cast<const uint32_t*>(src);
                    }
#pragma unroll
                    for (int e = 0; e < N / 2; ++e) {
                        const __nv_fp8x2_storage_t h = static_cast<__nv_fp8x2_storage_t>(q[e / 2] >> (16 * (e & 1)));
                        const float2 f = __half22float2(static_cast<__half2>(__nv_cvt_fp8x2_to_halfraw2(h, __NV_E4M3)));
                        x[k][e] = make_float2(f.x * sc, f.y * sc);
                    }
                } else {
                    Pc::load(static_cast<const T*>(p.x) + rr * p.xs + v * N, x[k]);
                }
            }
        }
        const float r = live ? p.rstd[rr] : 0.0f;
        float gn = 0.0f, none = 0.0f;
#pragma unroll
        for (int k = 0; k < NP; ++k) {
            const int v = l0 + k * step;
            float2 w[N / 2];
#pragma unroll
            for (int e = 0; e < N / 2; ++e) w[e] = splat2(0.0f);
            if (v < nvec) Pc::load_w(p.w + v * N, w);
#pragma unroll
            for (int e = 0; e < N / 2; ++e) {
                x[k][e] = fmul2(x[k][e], splat2(r));  // n
                dw[k][e] = ffma2(g[k][e], x[k][e], dw[k][e]);
                g[k][e] = fmul2(g[k][e], w[e]);
                gn = fmaf(g[k][e].x, x[k][e].x, fmaf(g[k][e].y, x[k][e].y, gn));
            }
        }
        row_sums(gn, none, p.wpr, s_red);
        const float m = -gn * p.inv_c;
        T* out = static_cast<T*>(p.out) + rr * p.C;
#pragma unroll
        for (int k = 0; k < NP; ++k) {
            const int v = l0 + k * step;
            if (live && v < nvec) {
                float2 o[N / 2];
#pragma unroll
                for (int e = 0; e < N / 2; ++e) o[e] = fmul2(ffma2(x[k][e], splat2(m), g[k][e]), splat2(r));
                Pc::store(out + v * N, o);
            }
        }
    }
    // the block's rows, one after another in a fixed order
    for (int s = 0; s < rpb; ++s) {
        if (sub == s) {
#pragma unroll
            for (int k = 0; k < NP; ++k) {
                const int v = l0 + k * step;
                if (v < nvec) {
#pragma unroll
                    for (int e = 0; e < N / 2; ++e) {
                        float2* d = reinterpret_cast<float2*>(s_dw + v * N) + e;
                        *d = s == 0 ? dw[k][e] : fadd2(*d, dw[k][e]);
                    }
                }
            }
        }
        __syncthreads();
    }
    float* part = p.part + int64_t(blockIdx.x) * p.C;
    for (int c = threadIdx.x; c < p.C; c += blockDim.x) part[c] = s_dw[c];
}

// ------------------------------------------------------------------ column sums
constexpr int kSumY = 16;
__global__ void __launch_bounds__(32 * kSumY) column_sums_kernel(const float* part, int64_t rows, int64_t C, float* out) {
    __shared__ float s[kSumY][32];
    const int64_t c = int64_t(blockIdx.x) * 32 + threadIdx.x;
    float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if (c < C) {
        int64_t r = threadIdx.y;
        for (; r + 3 * kSumY < rows; r += 4 * kSumY)
#pragma unroll
            for (int k = 0; k < 4; ++k) acc[k] += part[(r + k * kSumY) * C + c];
        for (int k = 0; r < rows; r += kSumY, ++k) acc[k] += part[r * C + c];
    }
    s[threadIdx.y][threadIdx.x] = (acc[0] + acc[1]) + (acc[2] + acc[3]);
    __syncthreads();
    if (threadIdx.y == 0 && c < C) {
        float t = 0.0f;
#pragma unroll
        for (int k = 0; k < kSumY; ++k) t += s[k][threadIdx.x];
        out[c] = t;
    }
}

// ------------------------------------------------------------------ launch
struct NormPlan {
    int np, wpr, rpb;
};
NormPlan norm_plan(int64_t nvec) {
    NormPlan pl{1, 1, 8};
    while (int64_t(pl.np) * 32 < nvec && pl.np < kPieces) pl.np *= 2;
    while (int64_t(pl.np) * 32 * pl.wpr < nvec) pl.wpr *= 2;
    pl.rpb = std::max(1, 8 / pl.wpr);
    return pl;
}
// Blocks of the backward: enough to fill the device, few enough that the
// partial rows they leave are a small part of the traffic.
constexpr int kBwdBlocks = 148 * 3;
int64_t bwd_blocks(int64_t rows, const NormPlan& pl) {
    return std::max<int64_t>(1, std::min<int64_t>(kBwdBlocks, (rows + pl.rpb - 1) / pl.rpb));
}

template <typename T, bool CK>
int launch_norm(bool bwd, const NormPlan& pl, const NormTrainParams& p, cudaStream_t s) {
    const int threads = 32 * pl.wpr * pl.rpb;
    const int64_t blocks = bwd ? bwd_blocks(p.rows, pl) : (p.rows + pl.rpb - 1) / pl.rpb;
    if (blocks > INT32_MAX) return fail(NEED_ERR_UNSUPPORTED, "rms norm: too many rows");
    const unsigned grid = static_cast<unsigned>(blocks);
    const size_t sm = bwd ? size_t(p.C) * 4 : 0;
    auto go = [&](auto np) {
        constexpr int NP = decltype(np)::value;
        if (bwd) {
            if (sm > 48 * 1024) {
                static std::atomic<uint64_t> done{0};
                const cudaError_t e = ensure_smem(norm_train_bwd<T, CK, NP>, 64 * 1024, done);
                if (e != cudaSuccess) return cuda_fail(e, "cudaFuncSetAttribute(norm_train_bwd)");
            }
            norm_train_bwd<T, CK, NP><<<grid, threads, sm, s>>>(p);
        } else {
            norm_train_fwd<T, CK, NP><<<grid, threads, 0, s>>>(p);
        }
        const cudaError_t e = cudaGetLastError();
        return e == cudaSuccess ? int(NEED_OK) : cuda_fail(e, "rms norm training launch");
    };
    if (pl.np == 1) return go(std::integral_constant<int, 1>{});
    if (pl.np == 2) return go(std::integral_constant<int, 2>{});
    return go(std::integral_constant<int, 4>{});
}

int norm_train(const need_norm_train_args* a, bool bwd, cudaStream_t s) {
    if (a == nullptr) return fail(NEED_ERR_INVALID, "args is null");
    if (!dtype_ok(a->dtype)) return fail(NEED_ERR_UNSUPPORTED, "rms norm: dtype %d", a->dtype);
    if (a->rows < 1 || a->C < 1) return fail(NEED_ERR_INVALID, "rms norm: sizes must be >= 1");
    const int64_t vec = 16 / dtype_bytes(a->dtype);
    if (a->C % vec != 0 || a->C / vec > int64_t(kMaxWarps) * 32 * kPieces)
        return fail(NEED_ERR_UNSUPPORTED, "rms norm: C=%lld must be a multiple of %lld and at most %lld",
                    (long long)a->C, (long long)vec, (long long)(vec * kMaxWarps * 32 * kPieces));
    if (a->C_mean < 1 || a->C_mean > a->C) return fail(NEED_ERR_INVALID, "rms norm: C_mean=%lld", (long long)a->C_mean);
    if (!(a->eps >= 0.0)) return fail(NEED_ERR_INVALID, "rms norm: eps must be >= 0");
    if (a->checkpoint != 0 && a->checkpoint != 1) return fail(NEED_ERR_INVALID, "checkpoint %d", a->checkpoint);
    if (a->checkpoint != 0 && (a->ckpt_values == nullptr || a->ckpt_scales == nullptr ||
                               reinterpret_cast<uintptr_t>(a->ckpt_values) % 8 != 0))
        return fail(NEED_ERR_INVALID, "rms norm: the 8-bit checkpoint is null or not 8-byte aligned");
    if (a->weight == nullptr || !aligned16(a->weight) || a->rstd == nullptr)
        return fail(NEED_ERR_INVALID, "rms norm: weight (16-byte aligned) and rstd must be non-null");
    const bool need_x = !bwd || a->checkpoint == 0;
    if (need_x && (a->x == nullptr || !aligned16(a->x) || (a->rows > 1 && a->x_stride % vec != 0)))
        return fail(NEED_ERR_UNSUPPORTED, "rms norm: x needs 16-byte aligned rows");
    if (bwd && (a->gout == nullptr || !aligned16(a->gout) || (a->rows > 1 && a->gout_stride % vec != 0)))
        return fail(NEED_ERR_UNSUPPORTED, "rms norm: gout needs 16-byte aligned rows");
    void* out = bwd ? a->grad_x : a->out;
    if (out == nullptr || !aligned16(out)) return fail(NEED_ERR_INVALID, "rms norm: the output is null or not 16-byte aligned");
    if (bwd && a->grad_weight == nullptr) return fail(NEED_ERR_INVALID, "rms norm: grad_weight is null");
    const NormPlan pl = norm_plan(a->C / vec);
    if (bwd && (a->workspace == nullptr || a->workspace_bytes < need_rms_norm_train_workspace_size(a->rows, a->C)))
        return fail(NEED_ERR_WORKSPACE, "rms norm: workspace missing or too small");
    NormTrainParams p{};
    p.x = a->x, p.xs = a->x_stride, p.gout = a->gout, p.gs = a->gout_stride, p.w = a->weight, p.out = out;
    p.rstd = a->rstd, p.q = a->ckpt_values, p.qs = a->ckpt_scales, p.part = static_cast<float*>(a->workspace);
    p.rows = a->rows, p.C = int32_t(a->C), p.ngroups = int32_t((a->C + kGroup - 1) / kGroup), p.wpr = pl.wpr;
    p.inv_c = 1.0f / static_cast<float>(a->C_mean), p.eps = static_cast<float>(a->eps);
    auto run = [&](auto tag) {
        using T = decltype(tag);
        return a->checkpoint != 0 ? launch_norm<T, true>(bwd, pl, p, s) : launch_norm<T, false>(bwd, pl, p, s);
    };
    int rc;
    if (a->dtype == NEED_F32) rc = run(float{});
    else if (a->dtype == NEED_BF16) rc = run(__nv_bfloat16{});
    else rc = run(__half{});
    if (rc == NEED_OK && bwd) rc = column_sums(p.part, bwd_blocks(a->rows, pl), a->C, a->grad_weight, s);
    return rc != NEED_OK ? rc : ok();
}

}  // namespace

namespace need {
int column_sums(const float* part, int64_t rows, int64_t C, float* out, cudaStream_t stream) {
    const unsigned grid = static_cast<unsigned>((C + 31) / 32);
    column_sums_kernel<<<grid, dim3(32, kSumY), 0, stream>>>(part, rows, C, out);
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? NEED_OK : cuda_fail(e, "column_sums_kernel launch");
}
}  // namespace need

extern "C" {

size_t need_rms_norm_train_workspace_size(int64_t rows, int64_t C) {
    if (rows < 1 || C < 1) return 16;
    return size_t(std::min<int64_t>(kBwdBlocks, rows)) * size_t(C) * 4;
}
int need_rms_norm_train_forward(const need_norm_train_args* args, need_stream_t stream) {
    return norm_train(args, false, stream);
}
int need_rms_norm_train_backward(const need_norm_train_args* args, need_stream_t stream) {
    return norm_train(args, true, stream);
}

}  // extern "C"
