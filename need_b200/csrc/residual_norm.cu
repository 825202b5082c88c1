// residual_norm.cu -- the residual's addition and the RMSNorm of what it gives, with an
// output in the row's type or in 8 bits with scales (need_residual_rms_norm):
//
//   r = x + scale y (rounded, the stream that goes on),  n = r / sqrt(sum(r^2) / C + eps) w
//   out = n, or e4m3(n / 2^e) with one 2^e for each `group` channels
//
// x and y are read once, the stream and the output written once: 8 B per 16-bit element,
// 7 with 8 bits, so HBM bounds it.  A row lies in the registers of 1 to 16 warps, from the
// addition to the output; its sum and the groups' largest values are taken by shuffles, a
// group's pieces lying in neighbouring lanes.  16384 rows of 832 bf16 channels: 17.0 us, 6.4
// TB/s; with 8 bits 20.3 us, 4.8 TB/s, by its instructions; 64 rows: 2.4 us, a launch and two
// round trips.  Rows that only 8, 4 or 2 bytes divide: 14288 rows of 1324 bf16 channels 27
// us, of 1326 43, of 1325 112.
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
constexpr int kRowBytes = kMaxWarps * 32 * kPieces * 16;

struct ResidualParams {
    const void* x;
    int64_t xs;
    const void* y;
    int64_t ys;
    const float* w;
    void* stream;
    int64_t ss;
    void* out;
    int64_t os;
    float* scales;
    int64_t rows;
    int32_t C, wpr, group, ngroups;  // group: of an 8-bit output; C for one scale a row
    float inv_c, eps, scale;
};

template <int BYTES>
struct Word;
template <>
struct Word<16> { using W = uint4; };
template <>
struct Word<8> { using W = uint2; };
template <>
struct Word<4> { using W = unsigned int; };
template <>
struct Word<2> { using W = unsigned short; };
template <>
struct Word<1> { using W = unsigned char; };

// A 16-byte piece of a row, M elements at a time, of which the first n are inside the row: M
// divides the channels, and M elements are what every row is aligned to.
template <typename T, int M>
__device__ __forceinline__ uint4 load_piece(const T* p, int n) {
    using W = typename Word<M * sizeof(T)>::W;
    constexpr int N = 16 / sizeof(T);
    union { uint4 u; W w[N / M]; } r;
    r.u = make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int e = 0; e < N; e += M)
        if (M == N || e < n) r.w[e / M] = __ldcs(reinterpret_cast<const W*>(p + e));
    return r.u;
}
// B: bytes of an element in memory
template <int B, int N, int M, typename U>
__device__ __forceinline__ void store_piece(void* p, int n, const U& u) {
    using W = typename Word<M * B>::W;
#pragma unroll
    for (int e = 0; e < N; e += M)
        if (M == N || e < n) reinterpret_cast<W*>(p)[e / M] = reinterpret_cast<const W*>(&u)[e / M];
}

// The larger of a (at least 0) and |b|; NaN if one of them is.
__device__ __forceinline__ float max_abs(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(fabsf(b)));
    return r;
}
// The weights of a piece's N channels, of which the first n are there.
template <int M, int N>
__device__ __forceinline__ void load_weights(const float* w, int n, float (&f)[N]) {
    constexpr int F = M < 4 ? M : 4;
    using W = typename Word<4 * F>::W;
#pragma unroll
    for (int e = 0; e < N; e += F) {
        union { W u; float f[F]; } r;
#pragma unroll
        for (int i = 0; i < F; ++i) r.f[i] = 0.0f;
        if (M == N || e < n) r.u = __ldg(reinterpret_cast<const W*>(w + e));
#pragma unroll
        for (int i = 0; i < F; ++i) f[e + i] = r.f[i];
    }
}

// blockDim = 32 * wpr * (rows per block); lane l of a row's warp w holds pieces
// (w * 32 + l) + k * 32 * wpr.  OUT8: the output in 8 bits.
template <typename T, int NP, int M, bool OUT8>
__global__ void __launch_bounds__(512) residual_norm_kernel(const ResidualParams p) {
    using P = typename Ops<T>::P;
    constexpr int N = 16 / Ops<T>::BYTES;
    __shared__ float s_red[kMaxWarps];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, w0 = warp / p.wpr * p.wpr;
    const int rpb = (blockDim.x >> 5) / p.wpr;
    const int64_t row = int64_t(blockIdx.x) * rpb + warp / p.wpr;
    const bool live = row < p.rows;
    const int l0 = (warp % p.wpr) * 32 + lane, step = 32 * p.wpr, nvec = (p.C + N - 1) / N;
    const T* x = static_cast<const T*>(p.x) + (live ? row : 0) * p.xs;
    const T* y = static_cast<const T*>(p.y) + (live ? row : 0) * p.ys;
    uint4 u[NP], v[NP];
#pragma unroll
    for (int k = 0; k < NP; ++k) {
        const int i = l0 + k * step;
        u[k] = v[k] = make_uint4(0, 0, 0, 0);
        if (live && i < nvec) u[k] = load_piece<T, M>(x + i * N, p.C - i * N), v[k] = load_piece<T, M>(y + i * N, p.C - i * N);
    }
    // the weights meanwhile, where a lane has at most 16: 64 rows of 832 fp32 channels 2.8 us,
    // 3.6 with them after the sum; at 32 of them they push rows out of the registers (16384
    // rows of 832 bf16 channels 18.7 us, 16.9 after the sum)
    constexpr bool EARLY = NP * N <= 16;
    float w[NP][N] = {};
    auto weights = [&](int k) {
        const int i = l0 + k * step;
        if (live && i < nvec) load_weights<M>(p.w + i * N, p.C - i * N, w[k]);
    };
#pragma unroll
    for (int k = 0; k < NP; ++k)
        if (EARLY) weights(k);
    float2 ss2 = make_float2(0.0f, 0.0f);
#pragma unroll
    for (int k = 0; k < NP; ++k) {
        P* a = reinterpret_cast<P*>(&u[k]);
        const P* b = reinterpret_cast<const P*>(&v[k]);
#pragma unroll
        for (int e = 0; e < N / 2; ++e) {
            const float2 r = ffma2(widen(b[e]), splat2(p.scale), widen(a[e]));
            a[e] = Ops<T>::pack(r.x, r.y);
            const float2 f = widen(a[e]);  // the stream as it goes on
            ss2 = ffma2(f, f, ss2);
        }
        const int i = l0 + k * step;
        if (live && i < nvec) store_piece<sizeof(T), N, M>(static_cast<T*>(p.stream) + row * p.ss + i * N, p.C - i * N, u[k]);
    }
    float ss = ss2.x + ss2.y;
#pragma unroll
    for (int m = 16; m >= 1; m >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, m);
    if (p.wpr > 1) {
        if (lane == 0) s_red[warp] = ss;
        __syncthreads();
        ss = 0.0f;
        for (int w = 0; w < p.wpr; ++w) ss += s_red[w0 + w];
    }
    const float inv = rsqrtf(fmaf(ss, p.inv_c, p.eps));

    if constexpr (!OUT8) {
#pragma unroll
        for (int k = 0; k < NP; ++k) {
            const int i = l0 + k * step;
            if (!live || i >= nvec) continue;
            P* a = reinterpret_cast<P*>(&u[k]);
            if (!EARLY) weights(k);
#pragma unroll
            for (int e = 0; e < N / 2; ++e) {
                const float2 f = fmul2(fmul2(widen(a[e]), splat2(inv)), make_float2(w[k][2 * e], w[k][2 * e + 1]));
                a[e] = Ops<T>::pack(f.x, f.y);
            }
            store_piece<sizeof(T), N, M>(static_cast<T*>(p.out) + row * p.os + i * N, p.C - i * N, u[k]);
        }
    } else {
        // n in fp32, and the largest magnitudes (a NaN above an infinity).  Places outside the
        // row are 0 here, and under a weight of 0: in a row without NaN they stay 0
        float2 n[NP][N / 2];
        float top[NP], most = 0.0f;
#pragma unroll
        for (int k = 0; k < NP; ++k) {
            const P* a = reinterpret_cast<const P*>(&u[k]);
            if (!EARLY) weights(k);
            top[k] = 0.0f;
#pragma unroll
            for (int e = 0; e < N / 2; ++e) {
                n[k][e] = fmul2(fmul2(widen(a[e]), splat2(inv)), make_float2(w[k][2 * e], w[k][2 * e + 1]));
                top[k] = max_abs(max_abs(top[k], n[k][e].x), n[k][e].y);
            }
            most = max_abs(most, top[k]);
        }
        uint32_t all = __float_as_uint(most);
        if (p.group == p.C) {  // one scale a row
            all = __reduce_max_sync(0xffffffffu, all);
            if (p.wpr > 1) {
                __syncthreads();  // the sums have been read
                if (lane == 0) s_red[warp] = __uint_as_float(all);
                __syncthreads();
                for (int w = 0; w < p.wpr; ++w) all = max(all, __float_as_uint(s_red[w0 + w]));
            }
        }
        const int lanes = p.group / N;  // that share a scale
#pragma unroll
        for (int k = 0; k < NP; ++k) {
            const int i = l0 + k * step;
            uint32_t t = all;
            if (p.group != p.C) {
                t = __float_as_uint(top[k]);
                for (int m = 1; m < lanes; m <<= 1) t = max(t, __shfl_xor_sync(0xffffffffu, t, m));
            }
            const uint32_t byte = e4m3_scale_byte(t);
            if (!live || i >= nvec) continue;
            const bool first = p.group != p.C ? (i & (lanes - 1)) == 0 : i == 0;
            if (first) p.scales[row * p.ngroups + (p.group != p.C ? i / lanes : 0)] = e4m3_scale(byte);
            alignas(N) uint16_t q[N / 2];
#pragma unroll
            for (int e = 0; e < N / 2; ++e) q[e] = e4m3_pair(n[k][e], byte);
            store_piece<1, N, M>(static_cast<uint8_t*>(p.out) + row * p.os + i * N, p.C - i * N, q);
        }
    }
}

template <typename T, int NP, int M>
int launch(const ResidualParams& p, bool out8, cudaStream_t s) {
    const int warps = std::max(p.wpr, 4), rpb = warps / p.wpr;
    const int64_t blocks = (p.rows + rpb - 1) / rpb;
    if (out8) residual_norm_kernel<T, NP, M, true><<<static_cast<unsigned>(blocks), 32 * warps, 0, s>>>(p);
    else residual_norm_kernel<T, NP, M, false><<<static_cast<unsigned>(blocks), 32 * warps, 0, s>>>(p);
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? NEED_OK : cuda_fail(e, "residual norm launch");
}

}  // namespace

extern "C" int need_residual_rms_norm(const need_residual_norm_args* a, need_stream_t stream) {
    if (a == nullptr) return fail(NEED_ERR_INVALID, "residual norm: args is null");
    if (!dtype_ok(a->dtype)) return fail(NEED_ERR_UNSUPPORTED, "residual norm: dtype %d", a->dtype);
    if (a->rows < 1 || a->C < 1) return fail(NEED_ERR_INVALID, "residual norm: sizes must be positive");
    const int es = dtype_bytes(a->dtype), n = 16 / es;
    if (a->C * es > kRowBytes || a->rows > (int64_t(1) << 31) - 1)
        return fail(NEED_ERR_UNSUPPORTED, "residual norm: rows of at most %d bytes, 2^31 - 1 of them", kRowBytes);
    if (!(a->eps >= 0.0)) return fail(NEED_ERR_INVALID, "residual norm: eps must be >= 0");
    if (a->x == nullptr || a->y == nullptr || a->weight == nullptr || a->stream == nullptr || a->out == nullptr)
        return fail(NEED_ERR_INVALID, "residual norm: x, y, weight, stream and out are required");
    if (a->out8 != 0 && (a->out8 != 1 || a->scales == nullptr || (a->group != 32 && a->group != 64 && a->group != 128 && a->group != a->C)))
        return fail(NEED_ERR_INVALID, "residual norm: an 8-bit output needs scales, one for 32, 64, 128 or all channels");
    if (a->rows > 1 && (a->stream_stride < a->C || a->out_stride < a->C))
        return fail(NEED_ERR_INVALID, "residual norm: the outputs' rows overlap");
    ResidualParams p{};
    p.x = a->x, p.xs = a->x_stride, p.y = a->y, p.ys = a->y_stride, p.w = a->weight;
    p.stream = a->stream, p.ss = a->stream_stride, p.out = a->out, p.os = a->out_stride, p.scales = a->scales;
    p.rows = a->rows, p.C = int32_t(a->C), p.group = a->out8 ? int32_t(a->group) : 0;
    p.ngroups = a->out8 ? int32_t((a->C + a->group - 1) / a->group) : 0;
    p.inv_c = 1.0f / static_cast<float>(a->C), p.eps = static_cast<float>(a->eps), p.scale = static_cast<float>(a->scale);
    const int nvec = int32_t((a->C + n - 1) / n);
    p.wpr = 1;
    // up to 2 MB of rows (which the GPU holds at once) a piece a lane, as far as the warps go:
    // 64 rows of 832 bf16 channels take 3.6 us at 4 pieces and 2.4 at one, 16384 17.0 and 20.1
    const int pieces = int64_t(a->rows) * a->C * es <= (2 << 20) ? 1 : kPieces;
    while (p.wpr * 32 * pieces < nvec && p.wpr < kMaxWarps) p.wpr *= 2;
    const int np = (nvec + 32 * p.wpr - 1) / (32 * p.wpr);
    // as many elements at a time as the channels divide into and every row is aligned to
    auto al = [&](const void* q, int64_t stride, int bytes, int m) {
        return reinterpret_cast<uintptr_t>(q) % (bytes * m) == 0 && (a->rows == 1 || stride % m == 0);
    };
    int m = n;
    while (m > 1 && !(a->C % m == 0 && al(a->weight, 0, 4, std::min(m, 4)) && al(p.x, p.xs, es, m) && al(p.y, p.ys, es, m) &&
                      al(p.stream, p.ss, es, m) && al(p.out, p.os, a->out8 ? 1 : es, m)))
        m /= 2;
    auto run = [&](auto tag) {
        using T = decltype(tag);
        auto go = [&](auto v) {
            constexpr int M = decltype(v)::value;
            switch (np) {
                case 1: return launch<T, 1, M>(p, a->out8 != 0, stream);
                case 2: return launch<T, 2, M>(p, a->out8 != 0, stream);
                case 3: return launch<T, 3, M>(p, a->out8 != 0, stream);
                default: return launch<T, 4, M>(p, a->out8 != 0, stream);
            }
        };
        if constexpr (sizeof(T) == 2)
            if (m == 8) return go(std::integral_constant<int, 8>{});
        if (m == 4) return go(std::integral_constant<int, 4>{});
        return m == 2 ? go(std::integral_constant<int, 2>{}) : go(std::integral_constant<int, 1>{});
    };
    const int rc = a->dtype == NEED_F32 ? run(float{}) : a->dtype == NEED_BF16 ? run(__nv_bfloat16{}) : run(__half{});
    return rc != NEED_OK ? rc : ok();
}
