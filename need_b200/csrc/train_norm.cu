// train_norm.cu -- RMSNorm with its gradient (need_rms_norm_train_forward,
// need_rms_norm_train_backward), the block's out_norm under training, and the
// fixed-order column sum the training kernels end with.
//
//   r = 1 / sqrt(sum(x^2) / C + eps), n = x r
//   y = n w;  g = w dy:  dx = r (g - n sum(g n) / C),  dw = sum over rows of dy n
//
// 4 B move per 16-bit element forward, 6 B backward, 5 and 5 with x kept in 8
// bits (8x2048x832 bf16: 11 us, 5.0 TB/s; 18 us, 4.5 TB/s, where 126 registers
// leave 16 warps an SM, each with its next row's loads in flight; 65536x1024: 112 us
// the pass, 6.0 TB/s).  A row is read once into the registers of 1 to 16 warps --
// the fewest that leave a lane at most 4 16-byte pieces -- and the two sums of the
// backward are reduced together.  The backward's blocks stride over the rows, so that
// a lane's channels stay the same and their share of dw stays in its registers, the
// next row's loads in flight while one is worked on; each block ends with one row of
// partial sums, and column_sums adds those rows in a fixed order.
#include <cuda_fp8.h>

#include <algorithm>
#include <type_traits>

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
    int64_t os;
    int64_t rows;
    int32_t C, ngroups, wpr;     // warps per row
    float inv_c, eps;
};

// Sums a over the warps of a row (all of them call it).
__device__ __forceinline__ float row_sum(float a, int wpr, float* s_red) {
#pragma unroll
    for (int m = 16; m >= 1; m >>= 1) a += __shfl_xor_sync(0xffffffffu, a, m);
    if (wpr > 1) {
        const int warp = threadIdx.x >> 5;
        __syncthreads();  // the previous row's sums have been read
        if ((threadIdx.x & 31) == 0) s_red[warp] = a;
        __syncthreads();
        const int w0 = warp / wpr * wpr;
        a = 0.0f;
        for (int w = 0; w < wpr; ++w) a += s_red[w0 + w];
    }
    return a;
}

// A 16-byte piece of a row, as loaded.  VEC: rows are 16-byte aligned and C whole
// pieces; else element by element, n of the piece's N elements inside C.
template <typename T, bool VEC>
struct Piece {
    using P = typename Ops<T>::P;
    static constexpr int N = 16 / Ops<T>::BYTES;
    static __device__ __forceinline__ uint4 load(const T* p, int n) {
        if constexpr (VEC) {
            return *reinterpret_cast<const uint4*>(p);
        } else {
            uint4 u;
            P* h = reinterpret_cast<P*>(&u);
#pragma unroll
            for (int e = 0; e < N / 2; ++e)
                h[e] = Ops<T>::pack(2 * e < n ? to_f(p[2 * e]) : 0.0f, 2 * e + 1 < n ? to_f(p[2 * e + 1]) : 0.0f);
            return u;
        }
    }
    static __device__ __forceinline__ void store(T* p, int n, const uint4& u) {
        if constexpr (VEC) {
            *reinterpret_cast<uint4*>(p) = u;
        } else {
            const T* q = reinterpret_cast<const T*>(&u);
            for (int e = 0; e < N && e < n; ++e) p[e] = q[e];
        }
    }
    static __device__ __forceinline__ void weights(const float* w, int n, float2 (&f)[N / 2]) {
        if constexpr (VEC) {
#pragma unroll
            for (int e = 0; e < N / 4; ++e) {
                const float4 q = __ldg(reinterpret_cast<const float4*>(w) + e);
                f[2 * e] = make_float2(q.x, q.y), f[2 * e + 1] = make_float2(q.z, q.w);
            }
        } else {
#pragma unroll
            for (int e = 0; e < N / 2; ++e)
                f[e] = make_float2(2 * e < n ? w[2 * e] : 0.0f, 2 * e + 1 < n ? w[2 * e + 1] : 0.0f);
        }
    }
};
template <typename T>
__device__ __forceinline__ float2 pair_of(const uint4& u, int e) {
    return widen(reinterpret_cast<const typename Ops<T>::P*>(&u)[e]);
}
template <typename T>
__device__ __forceinline__ void set_pair(uint4& u, int e, float2 f) {
    reinterpret_cast<typename Ops<T>::P*>(&u)[e] = Ops<T>::pack(f.x, f.y);
}

// blockDim = 32 * wpr * (rows per block); a row is handled by wpr warps, lane l
// of its warp w holding pieces (w * 32 + l) + k * 32 * wpr.
template <typename T, bool CK, int NP, bool VEC>
__global__ void __launch_bounds__(512) norm_train_fwd(const NormTrainParams p) {
    using Pc = Piece<T, VEC>;
    constexpr int N = Pc::N;
    __shared__ float s_red[kMaxWarps];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rpb = (blockDim.x >> 5) / p.wpr;
    const int64_t row = int64_t(blockIdx.x) * rpb + warp / p.wpr;
    const bool live = row < p.rows;
    const int l0 = (warp % p.wpr) * 32 + lane, step = 32 * p.wpr, nvec = (p.C + N - 1) / N;
    const T* x = static_cast<const T*>(p.x) + (live ? row : 0) * p.xs;
    uint4 u[NP];
#pragma unroll
    for (int k = 0; k < NP; ++k) {
        const int v = l0 + k * step;
        u[k] = make_uint4(0, 0, 0, 0);
        if (live && v < nvec) u[k] = Pc::load(x + v * N, p.C - v * N);
    }
    float ss = 0.0f;
#pragma unroll
    for (int k = 0; k < NP; ++k)
#pragma unroll
        for (int e = 0; e < N / 2; ++e) {
            const float2 f = pair_of<T>(u[k], e);
            ss = fmaf(f.x, f.x, fmaf(f.y, f.y, ss));
        }
    ss = row_sum(ss, p.wpr, s_red);
    const float r = 1.0f / sqrtf(fmaf(ss, p.inv_c, p.eps));
    if (live && l0 == 0) p.rstd[row] = r;
    T* out = static_cast<T*>(p.out) + row * p.os;
#pragma unroll
    for (int k = 0; k < NP; ++k) {
        const int v = l0 + k * step;
        const bool in = live && v < nvec;
        if constexpr (CK) {
            // 64 channels lie in 64 / N neighbouring lanes
            uint32_t top = 0;
#pragma unroll
            for (int e = 0; e < N / 2; ++e) {
                const float2 f = pair_of<T>(u[k], e);
                top = max(top, max(__float_as_uint(f.x) & 0x7fffffffu, __float_as_uint(f.y) & 0x7fffffffu));
            }
#pragma unroll
            for (int m = kGroup / N / 2; m >= 1; m >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, m));
            if (in) {
                const uint32_t sc = e4m3_scale_byte(top);
                uint32_t q[N / 4];
#pragma unroll
                for (int e = 0; e < N / 4; ++e)
                    q[e] = e4m3_pair(pair_of<T>(u[k], 2 * e), sc) | uint32_t(e4m3_pair(pair_of<T>(u[k], 2 * e + 1), sc)) << 16;
                uint8_t* dst = p.q + row * p.ngroups * kGroup + v * N;
                if constexpr (N == 8) *reinterpret_cast<uint2*>(dst) = make_uint2(q[0], q[1]);
                else *reinterpret_cast<uint32_t*>(dst) = q[0];
                if (v % (kGroup / N) == 0) p.qs[row * p.ngroups + v * N / kGroup] = static_cast<uint8_t>(sc);
            }
        }
        if (in) {
            uint4 o;
            float2 w[N / 2];
            Pc::weights(p.w + v * N, p.C - v * N, w);
#pragma unroll
            for (int e = 0; e < N / 2; ++e)
                set_pair<T>(o, e, fmul2(fmul2(pair_of<T>(u[k], e), splat2(r)), w[e]));
            Pc::store(out + v * N, p.C - v * N, o);
        }
    }
}

// A row's pieces on their way: x (or its 8-bit values and scale) and gout.
template <int NP, bool CK>
struct RowIn {
    uint4 g[NP];
    uint4 x[CK ? 1 : NP];
    uint2 q[CK ? NP : 1];
    uint32_t sc[CK ? NP : 1];
    float r;
};

template <typename T, bool CK, int NP, bool VEC>
__global__ void __launch_bounds__(512) norm_train_bwd(const NormTrainParams p) {
    using Pc = Piece<T, VEC>;
    constexpr int N = Pc::N;
    __shared__ float s_red[kMaxWarps];
    extern __shared__ __align__(16) float s_dw[];  // [C rounded up to a piece]
    // the weights, [N / 4][nvec], so that a warp reads neighbouring 16 bytes (from
    // memory a piece's lie 4 N bytes apart: a pass of 4096x16384 bf16 160 us, 137 so)
    float4* s_w = reinterpret_cast<float4*>(s_dw + (p.C + N - 1) / N * N);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rpb = (blockDim.x >> 5) / p.wpr, sub = warp / p.wpr;
    const int l0 = (warp % p.wpr) * 32 + lane, step = 32 * p.wpr, nvec = (p.C + N - 1) / N;
    float2 dw[NP][N / 2];
#pragma unroll
    for (int k = 0; k < NP; ++k)
#pragma unroll
        for (int e = 0; e < N / 2; ++e) dw[k][e] = splat2(0.0f);
    RowIn<NP, CK> in;
    auto fetch = [&](int64_t row) {
        const bool live = row < p.rows;
        const T* go = static_cast<const T*>(p.gout) + row * p.gs;
        in.r = live ? p.rstd[row] : 0.0f;
#pragma unroll
        for (int k = 0; k < NP; ++k) {
            const int v = l0 + k * step;
            in.g[k] = make_uint4(0, 0, 0, 0);
            if constexpr (CK) in.q[k] = make_uint2(0, 0), in.sc[k] = 1;
            else in.x[k] = make_uint4(0, 0, 0, 0);
            if (live && v < nvec) {
                in.g[k] = Pc::load(go + v * N, p.C - v * N);
                if constexpr (CK) {
                    const uint8_t* src = p.q + row * p.ngroups * kGroup + v * N;
                    in.sc[k] = p.qs[row * p.ngroups + v * N / kGroup];
                    if constexpr (N == 8) in.q[k] = *reinterpret_cast<const uint2*>(src);
                    else in.q[k].x = *reinterpret_cast<const uint32_t*>(src);
                } else {
                    in.x[k] = Pc::load(static_cast<const T*>(p.x) + row * p.xs + v * N, p.C - v * N);
                }
            }
        }
    };
    const int64_t stride = int64_t(gridDim.x) * rpb;
    fetch(int64_t(blockIdx.x) * rpb + sub);
    for (int v = threadIdx.x; v < nvec; v += blockDim.x) {
        float2 w[N / 2];
        Pc::weights(p.w + v * N, p.C - v * N, w);
#pragma unroll
        for (int e = 0; e < N / 4; ++e) s_w[e * nvec + v] = make_float4(w[2 * e].x, w[2 * e].y, w[2 * e + 1].x, w[2 * e + 1].y);
    }
    auto weights = [&](int v, float2 (&w)[N / 2]) {
#pragma unroll
        for (int e = 0; e < N / 4; ++e) {
            const float4 q = s_w[e * nvec + v];
            w[2 * e] = make_float2(q.x, q.y), w[2 * e + 1] = make_float2(q.z, q.w);
        }
    };
    __syncthreads();
    for (int64_t base = int64_t(blockIdx.x) * rpb; base < p.rows; base += stride) {
        const int64_t row = base + sub;
        const RowIn<NP, CK> cur = in;
        if (base + stride < p.rows) fetch(row + stride);  // in flight while this row is worked on
        auto n_of = [&](int k, int e) {  // n = x rstd of a pair
            if constexpr (CK) {
                const uint32_t w = e / 2 == 0 ? cur.q[k].x : cur.q[k].y;
                const __nv_fp8x2_storage_t h = static_cast<__nv_fp8x2_storage_t>(w >> (16 * (e & 1)));
                const float2 f = __half22float2(static_cast<__half2>(__nv_cvt_fp8x2_to_halfraw2(h, __NV_E4M3)));
                return fmul2(fmul2(f, splat2(e4m3_scale(cur.sc[k]))), splat2(cur.r));
            } else {
                return fmul2(pair_of<T>(cur.x[k], e), splat2(cur.r));
            }
        };
        float gn = 0.0f;
#pragma unroll
        for (int k = 0; k < NP; ++k) {
            const int v = l0 + k * step;
            if (v < nvec) {
                float2 w[N / 2];
                weights(v, w);
#pragma unroll
                for (int e = 0; e < N / 2; ++e) {
                    const float2 n = n_of(k, e), go = pair_of<T>(cur.g[k], e);
                    const float2 gw = fmul2(go, w[e]);
                    dw[k][e] = ffma2(go, n, dw[k][e]);
                    gn = fmaf(gw.x, n.x, fmaf(gw.y, n.y, gn));
                }
            }
        }
        gn = row_sum(gn, p.wpr, s_red);
        const float2 m = splat2(-gn * p.inv_c), r2 = splat2(cur.r);
        T* out = static_cast<T*>(p.out) + row * p.os;
#pragma unroll
        for (int k = 0; k < NP; ++k) {
            const int v = l0 + k * step;
            if (row < p.rows && v < nvec) {
                uint4 o;
                float2 w[N / 2];
                weights(v, w);
#pragma unroll
                for (int e = 0; e < N / 2; ++e) {
                    const float2 gw = fmul2(pair_of<T>(cur.g[k], e), w[e]);
                    set_pair<T>(o, e, fmul2(ffma2(n_of(k, e), m, gw), r2));
                }
                Pc::store(out + v * N, p.C - v * N, o);
            }
        }
    }
    // the block's rows, one after another in a fixed order; a row's pieces follow each
    // other by a step, so that up to NP rows add at once
    for (int s = 0; s < rpb + NP - 1; ++s) {
#pragma unroll
        for (int k = 0; k < NP; ++k) {
            const int v = l0 + k * step;
            if (sub + k == s && v < nvec) {
                float4* d = reinterpret_cast<float4*>(s_dw + v * N);
#pragma unroll
                for (int e = 0; e < N / 4; ++e) {
                    const float2 a = dw[k][2 * e], b = dw[k][2 * e + 1];
                    const float4 o = sub == 0 ? make_float4(0.0f, 0.0f, 0.0f, 0.0f) : d[e];
                    d[e] = make_float4(o.x + a.x, o.y + a.y, o.z + b.x, o.w + b.y);
                }
            }
        }
        __syncthreads();
    }
    float* part = p.part + int64_t(blockIdx.x) * p.C;
    for (int c = threadIdx.x; c < p.C; c += blockDim.x) part[c] = s_dw[c];
}

// ------------------------------------------------------------------ column sums
// A block sums X columns, 512 / X threads a column.
constexpr int kSumThreads = 512;
constexpr int kSumRows = 4;   // rows a thread has on their way
template <int X>
__global__ void __launch_bounds__(kSumThreads) column_sums_kernel(const float* part, int64_t rows, int64_t C, float* out) {
    constexpr int Y = kSumThreads / X, W = kSumThreads / 32;
    __shared__ float s[W][X];
    const int x = threadIdx.x % X, lane = threadIdx.x & 31;
    const int64_t c = int64_t(blockIdx.x) * X + x;
    float acc[kSumRows] = {};
    if (c < C)
        for (int64_t r = threadIdx.x / X; r < rows; r += kSumRows * Y) {
            float v[kSumRows];
#pragma unroll
            for (int k = 0; k < kSumRows; ++k) v[k] = r + k * Y < rows ? part[(r + k * Y) * C + c] : 0.0f;
#pragma unroll
            for (int k = 0; k < kSumRows; ++k) acc[k] += v[k];
        }
    float t = (acc[0] + acc[1]) + (acc[2] + acc[3]);
#pragma unroll
    for (int m = X; m < 32; m *= 2) t += __shfl_xor_sync(0xffffffffu, t, m);
    if (lane < X) s[threadIdx.x >> 5][lane] = t;
    __syncthreads();
    if (threadIdx.x < X && c < C) {
        t = 0.0f;
#pragma unroll
        for (int w = 0; w < W; ++w) t += s[w][x];
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
// Blocks of the backward: as many as are resident at once where rows take up to 8 warps,
// so that blocks walk the same number of rows or one more (8x2048x832 bf16: 18 us; 23 us with 3
// per SM), and few enough that the partial rows they leave are a small part of the
// traffic.  Rows of 16 warps (past 16 KB) leave one block on an SM: two waves.
constexpr int kBwdBlocks = 148 * 2;
int64_t bwd_blocks(int64_t rows, const NormPlan& pl) {
    return std::max<int64_t>(1, std::min<int64_t>(kBwdBlocks, (rows + pl.rpb - 1) / pl.rpb));
}

template <typename T, bool CK, bool VEC>
int launch_norm(bool bwd, const NormPlan& pl, const NormTrainParams& p, cudaStream_t s) {
    const int threads = 32 * pl.wpr * pl.rpb;
    const int64_t blocks = bwd ? bwd_blocks(p.rows, pl) : (p.rows + pl.rpb - 1) / pl.rpb;
    if (blocks > INT32_MAX) return fail(NEED_ERR_UNSUPPORTED, "rms norm: too many rows");
    const unsigned grid = static_cast<unsigned>(blocks);
    const size_t sm = bwd ? 2 * (size_t(p.C + 7) / 8 * 8 * 4) : 0;
    auto go = [&](auto np) {
        constexpr int NP = decltype(np)::value;
        if (bwd) {
            if (sm + sizeof(float) * kMaxWarps > 48 * 1024) {  // with the kernel's static shared memory
                static std::atomic<uint64_t> done{0};
                const cudaError_t e = ensure_smem(norm_train_bwd<T, CK, NP, VEC>, 128 * 1024, done);
                if (e != cudaSuccess) return cuda_fail(e, "cudaFuncSetAttribute(norm_train_bwd)");
            }
            norm_train_bwd<T, CK, NP, VEC><<<grid, threads, sm, s>>>(p);
        } else {
            norm_train_fwd<T, CK, NP, VEC><<<grid, threads, 0, s>>>(p);
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
    if (a->C > vec * kMaxWarps * 32 * kPieces)
        return fail(NEED_ERR_UNSUPPORTED, "rms norm: C=%lld, at most %lld", (long long)a->C,
                    (long long)(vec * kMaxWarps * 32 * kPieces));
    if (!(a->eps >= 0.0)) return fail(NEED_ERR_INVALID, "rms norm: eps must be >= 0");
    if (a->checkpoint != 0 && a->checkpoint != 1) return fail(NEED_ERR_INVALID, "checkpoint %d", a->checkpoint);
    if (a->checkpoint != 0 && (a->ckpt_values == nullptr || a->ckpt_scales == nullptr ||
                               reinterpret_cast<uintptr_t>(a->ckpt_values) % 8 != 0))
        return fail(NEED_ERR_INVALID, "rms norm: the 8-bit checkpoint is null or not 8-byte aligned");
    if (a->weight == nullptr || a->rstd == nullptr)
        return fail(NEED_ERR_INVALID, "rms norm: weight and rstd must be non-null");
    if ((!bwd || a->checkpoint == 0) && a->x == nullptr) return fail(NEED_ERR_INVALID, "rms norm: x is null");
    if (bwd && (a->gout == nullptr || a->grad_weight == nullptr))
        return fail(NEED_ERR_INVALID, "rms norm: gout and grad_weight must be non-null");
    void* out = bwd ? a->grad_x : a->out;
    if (out == nullptr) return fail(NEED_ERR_INVALID, "rms norm: the output is null");
    if (a->rows > 1 && a->out_stride < a->C) return fail(NEED_ERR_INVALID, "rms norm: the output's rows overlap");
    const NormPlan pl = norm_plan((a->C + vec - 1) / vec);
    if (bwd && (a->workspace == nullptr || a->workspace_bytes < need_rms_norm_train_workspace_size(a->rows, a->C)))
        return fail(NEED_ERR_WORKSPACE, "rms norm: workspace missing or too small");
    NormTrainParams p{};
    p.x = a->x, p.xs = a->x_stride, p.gout = a->gout, p.gs = a->gout_stride, p.w = a->weight;
    p.out = out, p.os = a->out_stride;
    auto al = [&](const void* q, int64_t stride) { return aligned16(q) && (a->rows == 1 || stride % vec == 0); };
    const bool whole = a->C % vec == 0 && al(p.out, p.os) && al(p.w, 0) && (bwd ? al(p.gout, p.gs) : true) &&
                       (bwd && a->checkpoint != 0 ? true : al(p.x, p.xs));
    p.rstd = a->rstd, p.q = a->ckpt_values, p.qs = a->ckpt_scales, p.part = static_cast<float*>(a->workspace);
    p.rows = a->rows, p.C = int32_t(a->C), p.ngroups = int32_t((a->C + kGroup - 1) / kGroup), p.wpr = pl.wpr;
    p.inv_c = 1.0f / static_cast<float>(a->C), p.eps = static_cast<float>(a->eps);
    auto run = [&](auto tag) {
        using T = decltype(tag);
        auto go = [&](auto ck) {
            constexpr bool CK = decltype(ck)::value;
            return whole ? launch_norm<T, CK, true>(bwd, pl, p, s) : launch_norm<T, CK, false>(bwd, pl, p, s);
        };
        return a->checkpoint != 0 ? go(std::true_type{}) : go(std::false_type{});
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
    // many rows of few columns: more threads a column (256x832: 2.7 us against 3.4), elsewhere
    // whole 128-byte lines (296x16384: a pass of the norm 137 us against 144)
    if (rows > 64 && C <= 32 * 74)
        column_sums_kernel<8><<<static_cast<unsigned>((C + 7) / 8), kSumThreads, 0, stream>>>(part, rows, C, out);
    else
        column_sums_kernel<32><<<static_cast<unsigned>((C + 31) / 32), kSumThreads, 0, stream>>>(part, rows, C, out);
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
