// linear_attention_umma.cu -- linear attention with a decay for each head on sm_100a's
// tensor cores (tcgen05): bf16, up to 128 features, rows of whole 16 bytes.  The
// mathematics, the planes and the segments are those of linear_attention.cu; the
// chunks have 128 tokens.
//
// One CTA walks the chunks of one (sequence, head, 64 columns of v).  Per chunk, with
// fp32 accumulators in tensor memory:
//
//   P    = Q K^T                 128 x 128          (two buffers)
//   O2   = Q S                   128 x 64           S: 2 planes, shared memory
//   O1   = P' V                  128 x 64           P' = P with its decays, 2 planes, in P's place
//   dS^T = (V w)^T K             64 x features      V w: 3 planes, shared memory
//   out  = O1 + e^G O2,  S' = e^{G_end} S + dS
//
// The state lies in the registers of the warps that add dS to it.  Each kind of work has
// warps of its own, which meet at mbarriers only, so that a chunk's scores, outputs and
// state run beside its neighbours':
//
//   warps 0-3    P'    a row per thread; below the diagonal's blocks a decay is a row's factor
//                      times a column's, so that only the blocks on it take an exponential
//                      per score
//   warps 4-7    V w, the state and its planes, the check for infinities
//   warps 8-11   outputs
//   warp 12      one lane: TMA loads (no multicast) and all MMAs
//   warp 13      the decays of the chunks ahead
//
// Every wait is bounded.  A block that gave one up, or met a value that is not finite (or
// a log decay that makes a chunk's products leave fp32's range), says so in `redo`:
// attention_kernel, launched behind, then computes the block's whole segment.
#include <cuda.h>
#include <cuda_bf16.h>

#include <algorithm>

#include "host_common.h"
#include "linear_attention.cuh"
#include "need_scan.h"
#include "ptx.cuh"
#include "umma.cuh"

using namespace need;
using namespace need::attention;

namespace {

constexpr int CT = 128;      // tokens of a chunk
constexpr int DVS = 64;      // columns of v of a CTA
constexpr int kThreads = 448;
constexpr int GR = 4;        // chunks whose decays are held
constexpr uint32_t kPolls = 1u << 18;  // of a wait before it is given up
constexpr uint32_t kTmem = 512, T_P = 0, T_O1 = 256, T_O2 = 320, T_DS = 384;  // tensor memory columns
constexpr int kVPlanes = 3;

struct alignas(16) Gates {
    float hi[CT], lo[CT], w[CT], eg[CT], end[CT];  // as Decays; end: of its block of 32
    int seg[CT];
    float d;
    int wild;
};

template <int DK>
struct Map {  // shared memory, from a 1024-byte aligned base
    static constexpr int NQ = DK == 64 ? 2 : 1, NK = DK == 64 ? 3 : 2, NV = NK;  // chunks loaded ahead
    static constexpr int QB = CT * DK * 2, VB = CT * DVS * 2, SB = DVS * DK * 2;
    static constexpr int Q = 0, K = Q + NQ * QB, V = K + NK * QB, W = V + NV * VB, S = W + kVPlanes * VB, G = S + 2 * SB;
    static constexpr int BAR = G + GR * static_cast<int>(sizeof(Gates)), BYTES = BAR + 512 + 1024;
};

struct UmmaParams {
    CUtensorMap q, k, v;  // [sequence, token, head, feature], boxes of 128 tokens x 64 features
    AttnParams a;
    uint32_t* redo;
    uint32_t polls;
};

__device__ __forceinline__ void tma_load(uint32_t dst, const CUtensorMap* tm, int c0, int c1, int c2, int c3, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst), "l"(tm), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(smem_addr(bar))
        : "memory");
}
// D[tmem] (+)= A[tmem] B[smem]
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(idesc),
        "r"(accumulate ? 1u : 0u)
        : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t (&v)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
        "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
        "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
        "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]),
        "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]), "r"(v[19]), "r"(v[20]),
        "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]), "r"(v[28]), "r"(v[29]), "r"(v[30]),
        "r"(v[31])
        : "memory");
}
// 64 columns of 16 lanes: the four values of 8 columns lie as in a 16 x 8 accumulator of
// mma.sync (rows lane / 4 and + 8, columns 2 (lane % 4) and + 1).
__device__ __forceinline__ void tmem_ld16x64(uint32_t taddr, float (&v)[32]) {
    uint32_t r[32];
    asm volatile(
        "tcgen05.ld.sync.aligned.16x256b.x8.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
          "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]),
          "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
          "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr));
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}

// ------------------------------------------------------------------ decays
struct Tokens {  // a lane's 4 tokens of a chunk
    float ld[4];
    bool reset[4];
};
__device__ __forceinline__ Tokens load_tokens(const AttnParams& p, const float* ld, const uint8_t* seg, int64_t t0) {
    Tokens r;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const int64_t t = t0 + 4 * (threadIdx.x & 31) + e;
        const bool live = t < p.T;
        const float x = live ? ld[t * p.lt] : 0.0f;
        r.reset[e] = (live && seg != nullptr && seg[t * p.gt] != 0) || x == -INFINITY;
        r.ld[e] = r.reset[e] ? 0.0f : x < -10000.0f ? -10000.0f : x;  // a NaN stays one
    }
    return r;
}
__device__ __forceinline__ void make_gates(const Tokens& tp, float scale, Gates& g) {
    const int lane = threadIdx.x & 31;
    double G[4], sum = 0.0;
#pragma unroll
    for (int e = 0; e < 4; ++e) G[e] = sum += static_cast<double>(tp.ld[e]) * 1.4426950408889634074;
    double incl = sum;
#pragma unroll
    for (int m = 1; m < 32; m <<= 1) {
        const double o = __shfl_up_sync(0xffffffffu, incl, m);
        if (lane >= m) incl += o;
    }
    double before = __shfl_up_sync(0xffffffffu, incl, 1);
    if (lane == 0) before = 0.0;
    const uint32_t lt = (1u << lane) - 1u;
    int s = 0, send = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const uint32_t m = __ballot_sync(0xffffffffu, tp.reset[e]);
        s += __popc(m & lt), send += __popc(m);
    }
    const double end = __shfl_sync(0xffffffffu, incl, 31), block_end = __shfl_sync(0xffffffffu, incl, lane | 7);
    bool wild = false;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const int i = 4 * lane + e;
        const double x = before + G[e];
        const float hi = static_cast<float>(x);
        s += tp.reset[e] ? 1 : 0;
        g.hi[i] = hi, g.lo[i] = static_cast<float>(x - hi);
        g.seg[i] = s;
        g.w[i] = s == send ? ex2(static_cast<float>(end - x)) : 0.0f;
        g.eg[i] = s == 0 ? scale * ex2(hi) : 0.0f;
        g.end[i] = ex2(static_cast<float>(block_end - x));
        wild |= !(tp.ld[e] <= 0.5f);  // 128 of them stay below 2^93
    }
    wild = __any_sync(0xffffffffu, wild);
    if (lane == 0) g.d = send == 0 ? ex2(static_cast<float>(end)) : -1.0f, g.wild = wild ? 1 : 0;
}

// Whether one of 8 bf16 values is an infinity or NaN.
__device__ __forceinline__ void check8(const uint4& u, __nv_bfloat162& chk) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int e = 0; e < 4; ++e)
        chk = __hfma2(*reinterpret_cast<const __nv_bfloat162*>(&w[e]), __floats2bfloat162_rn(0.0f, 0.0f), chk);
}

// ------------------------------------------------------------------ the kernel
template <int DK, bool STATE>
__global__ void __launch_bounds__(kThreads, 1) umma_attention_kernel(const __grid_constant__ UmmaParams up) {
    using M = Map<DK>;
    constexpr int NQ = M::NQ, NK = M::NK, NV = M::NV, NI = DK / 8;
    const AttnParams& p = up.a;
    extern __shared__ unsigned char smem_raw[];
    unsigned char* const base = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const uint32_t sb = smem_addr(base);
    uint64_t* bar = reinterpret_cast<uint64_t*>(base + M::BAR);
    uint64_t *full_q = bar, *full_k = full_q + NQ, *full_v = full_k + NK, *gates_full = full_v + NV, *gates_free = gates_full + GR,
             *s_ready = gates_free + GR, *vw_ready = s_ready + 1, *qk_done = vw_ready + 1 /* 2 */, *ds_done = qk_done + 2,
             *p_ready = ds_done + 1 /* 2 */, *o_done = p_ready + 2, *o1_free = o_done + 1, *o2_free = o1_free + 1, *drain = o2_free + 1;
    uint32_t* const tbase = reinterpret_cast<uint32_t*>(drain + 1);
    volatile uint32_t* const dead = tbase + 1;
    uint32_t* const bad_word = tbase + 2;
    Gates* const gates = reinterpret_cast<Gates*>(base + M::G);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    int64_t id = blockIdx.x;
    const int nseg = STATE ? p.nseg - 1 : p.nseg;
    const int seg = static_cast<int>(id % nseg);
    id /= nseg;
    const int slice = static_cast<int>(id % p.slices);
    const int64_t chain = id / p.slices;
    const int b = static_cast<int>(chain / p.H), h = static_cast<int>(chain % p.H), col0 = slice * DVS;
    const int64_t first = int64_t(seg) * p.seg_chunks * 64;
    const int64_t last = first + int64_t(p.seg_chunks) * 64 < p.T ? first + int64_t(p.seg_chunks) * 64 : p.T;
    const int n = static_cast<int>((last - first + CT - 1) / CT);
    const float* ld = p.ld + b * p.lb + h * p.lh;
    const uint8_t* marks = p.seg == nullptr ? nullptr : p.seg + b * p.gb;

    if (threadIdx.x == 0) {
        for (uint64_t* x = full_q; x < gates_full; ++x) mbar_init(x, 1);
        for (int i = 0; i < GR; ++i) mbar_init(gates_full + i, 1), mbar_init(gates_free + i, STATE ? 4 : 12);
        mbar_init(s_ready, 4), mbar_init(vw_ready, 4), mbar_init(qk_done, 1), mbar_init(qk_done + 1, 1), mbar_init(ds_done, 1);
        mbar_init(p_ready, 4), mbar_init(p_ready + 1, 4), mbar_init(o_done, 1), mbar_init(o1_free, 4), mbar_init(o2_free, 4);
        mbar_init(drain, 1);
        *dead = 0, *bad_word = 0;
        fence_barrier_init();
    }
    if (warp == 12) {
        umma::tmem_alloc(tbase, kTmem);
        umma::tmem_relinquish();
    }
    umma::fence_before_sync();
    __syncthreads();
    umma::fence_after_sync();
    const uint32_t tmem = *tbase;
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;  // this warp's part of tensor memory

    // bounded; after one was given up nobody waits any more
    auto wait = [&](uint64_t* x, uint32_t phase) {
        for (uint32_t i = 0; i < up.polls; ++i) {
            if (mbar_try_wait(x, phase & 1u)) return;
            if (*dead) return;
        }
        *dead = 1;
    };
    auto arrive = [&](uint64_t* x) {  // one of a warp's lanes, for all
        __syncwarp();
        if (lane == 0) mbar_arrive(x);
    };

    if (warp < 4) {
        // ---------------------------------------------------------------- P'
        if constexpr (!STATE) {
            const int r = 32 * warp + lane;
            for (int c = 0; c < n; ++c) {
                const Gates& g = gates[c % GR];
                wait(gates_full + c % GR, c / GR);
                const float hr = g.hi[r], lr = g.lo[r];
                const int sr = g.seg[r];
                const bool resets = g.d == -1.0f;
                wait(qk_done + (c & 1), c >> 1);
                umma::fence_after_sync();
                const uint32_t tp = tmem + T_P + 128 * (c & 1) + lanes;
#pragma unroll 1
                for (int cb = 0; cb < 4; ++cb) {
                    uint32_t pl[32];  // the first planes of 32 scores, then the second
                    if (cb > warp) {
#pragma unroll
                        for (int e = 0; e < 32; ++e) pl[e] = 0u;
                    } else {
                        float x[32];
                        umma::tmem_ld32(tp + 32 * cb, x);
                        const bool pairwise = cb == warp || resets;
                        float f = 0.0f;
                        if (!pairwise) f = p.scale * ex2((hr - g.hi[32 * cb + 31]) + (lr - g.lo[32 * cb + 31]));
                        umma::tmem_wait_ld();
                        if (!pairwise) {
#pragma unroll
                            for (int e = 0; e < 32; e += 4) {
                                const float4 end = *reinterpret_cast<const float4*>(&g.end[32 * cb + e]);
                                const float2 a = __fmul2_rn(make_float2(x[e], x[e + 1]), __fmul2_rn(make_float2(end.x, end.y), splat(f)));
                                const float2 d = __fmul2_rn(make_float2(x[e + 2], x[e + 3]), __fmul2_rn(make_float2(end.z, end.w), splat(f)));
                                x[e] = a.x, x[e + 1] = a.y, x[e + 2] = d.x, x[e + 3] = d.y;
                            }
                        } else {
#pragma unroll
                            for (int e = 0; e < 32; e += 4) {
                                const float4 hs = *reinterpret_cast<const float4*>(&g.hi[32 * cb + e]);
                                const float4 ls = *reinterpret_cast<const float4*>(&g.lo[32 * cb + e]);
                                const int4 ss = *reinterpret_cast<const int4*>(&g.seg[32 * cb + e]);
                                const float hv[4] = {hs.x, hs.y, hs.z, hs.w}, lv[4] = {ls.x, ls.y, ls.z, ls.w};
                                const int sv[4] = {ss.x, ss.y, ss.z, ss.w};
#pragma unroll
                                for (int i = 0; i < 4; ++i)
                                    x[e + i] = sv[i] == sr && 32 * cb + e + i <= r ? x[e + i] * (p.scale * ex2((hr - hv[i]) + (lr - lv[i]))) : 0.0f;
                            }
                        }
#pragma unroll
                        for (int e = 0; e < 16; ++e) {
                            uint32_t two[2];
                            split<2>(make_float2(x[2 * e], x[2 * e + 1]), two);
                            pl[e] = two[0], pl[16 + e] = two[1];
                        }
                    }
                    tmem_st32(tp + 32 * cb, pl);
                }
                umma::tmem_wait_st();
                umma::fence_before_sync();
                arrive(p_ready + (c & 1));
                arrive(gates_free + c % GR);
            }
        }
    } else if (warp < 8) {
        // ---------------------------------------------------------------- V w and the state
        const int bw = warp - 4, bt = threadIdx.x - 128, gr = lane >> 2, c2 = (lane & 3) * 2, j0 = col0 + 16 * bw + gr;
        float s[NI][4];  // transposed: rows j0 and + 8, columns 8 n + c2 and + 1
        {
            const float* from = STATE ? nullptr : seg > 0 ? p.part + (chain * (p.nseg - 1) + seg - 1) * p.dk * int64_t(p.dv)
                                      : p.s0 != nullptr   ? p.s0 + chain * p.dk * int64_t(p.dv) : nullptr;
#pragma unroll
            for (int m = 0; m < NI; ++m)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int i = 8 * m + c2 + (e & 1), j = j0 + (e >> 1) * 8;
                    s[m][e] = from != nullptr && i < p.dk && j < p.dv ? from[int64_t(i) * p.dv + j] : 0.0f;
                }
        }
        auto publish = [&] {  // the state's planes, as the K-major B of Q S
#pragma unroll
            for (int m = 0; m < NI; ++m)
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    uint32_t two[2];
                    split<2>(make_float2(s[m][2 * r], s[m][2 * r + 1]), two);
#pragma unroll
                    for (int a = 0; a < 2; ++a)
                        *reinterpret_cast<uint32_t*>(base + M::S + a * M::SB + (m >> 3) * (DVS * 128) +
                                                     umma::sw128(16 * bw + gr + 8 * r, m & 7) + c2 * 2) = two[a];
                }
            fence_proxy_async_shared();
            arrive(s_ready);
        };
        if (!STATE) publish();
        float total = 1.0f;
        bool bad = false;
        for (int c = 0; c < n; ++c) {
            const Gates& g = gates[c % GR];
            wait(gates_full + c % GR, c / GR);
            wait(full_v + c % NV, c / NV);
            wait(full_k + c % NK, c / NK);
            const unsigned char *vt = base + M::V + (c % NV) * M::VB, *kt = base + M::K + (c % NK) * M::QB;
            __nv_bfloat162 chk = __floats2bfloat162_rn(0.0f, 0.0f);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int row = bt / 8 + 16 * i;
                const uint32_t off = umma::sw128(row, bt % 8);
                const uint4 u = *reinterpret_cast<const uint4*>(vt + off);
                check8(u, chk);
                const float2 w = splat(g.w[row]);
                const uint32_t x[4] = {u.x, u.y, u.z, u.w};
                uint32_t pl[4][kVPlanes];
#pragma unroll
                for (int e = 0; e < 4; ++e) split<kVPlanes>(__fmul2_rn(w, unpack_bf16(x[e])), pl[e]);
#pragma unroll
                for (int a = 0; a < kVPlanes; ++a)
                    *reinterpret_cast<uint4*>(base + M::W + a * M::VB + off) = make_uint4(pl[0][a], pl[1][a], pl[2][a], pl[3][a]);
            }
            fence_proxy_async_shared();
            umma::fence_before_sync();  // the last chunk's dS has been read
            arrive(vw_ready);
#pragma unroll
            for (int i = 0; i < DK / 8; ++i)
                check8(*reinterpret_cast<const uint4*>(kt + (i / 8) * (CT * 128) + umma::sw128(bt / 8 + 16 * (i % 8), bt % 8)), chk);
            const float2 f = __bfloat1622float2(chk);
            bad |= !(f.x == 0.0f && f.y == 0.0f) || g.wild != 0;
            const float d = g.d;
            total = total == -1.0f || d == -1.0f ? -1.0f : total * d;
            wait(ds_done, c);
            umma::fence_after_sync();
#pragma unroll
            for (int m0 = 0; m0 < NI; m0 += 8) {
                float x[32];
                tmem_ld16x64(tmem + T_DS + 8 * m0 + lanes, x);
                umma::tmem_wait_ld();
#pragma unroll
                for (int m = 0; m < 8; ++m)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        float& y = s[m0 + m][e];
                        y = d == -1.0f ? x[4 * m + e] : fmaf(d, y, x[4 * m + e]);
                    }
            }
            if (!STATE && c + 1 < n) publish();
            arrive(gates_free + c % GR);
        }
        if (bad) *bad_word = 1;
        float* const to = STATE ? p.part + (chain * (p.nseg - 1) + seg) * p.dk * int64_t(p.dv)
                                : seg == p.nseg - 1 && p.sT != nullptr ? p.sT + chain * p.dk * int64_t(p.dv) : nullptr;
        if (to != nullptr)
#pragma unroll
            for (int m = 0; m < NI; ++m)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int i = 8 * m + c2 + (e & 1), j = j0 + (e >> 1) * 8;
                    if (i < p.dk && j < p.dv) to[int64_t(i) * p.dv + j] = s[m][e];
                }
        if (STATE && slice == 0 && bt == 0) p.part_d[chain * (p.nseg - 1) + seg] = total;
    } else if (warp < 12) {
        // ---------------------------------------------------------------- outputs
        if constexpr (!STATE) {
            const int r = 32 * (warp - 8) + lane;
            __nv_bfloat16* const out = static_cast<__nv_bfloat16*>(p.out) + b * p.ob + h * p.oh + col0;
            for (int c = 0; c < n; ++c) {
                const Gates& g = gates[c % GR];
                wait(gates_full + c % GR, c / GR);
                const float eg = g.eg[r];
                const bool reach = g.seg[r] == 0;
                arrive(gates_free + c % GR);
                wait(qk_done + (c & 1), c >> 1);
                umma::fence_after_sync();
                float x[2][32];
                umma::tmem_ld32(tmem + T_O2 + lanes, x[0]);
                umma::tmem_ld32(tmem + T_O2 + 32 + lanes, x[1]);
                umma::tmem_wait_ld();
                umma::fence_before_sync();
                arrive(o2_free);
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int e = 0; e < 32; ++e) x[i][e] = reach ? eg * x[i][e] : 0.0f;
                wait(o_done, c);
                umma::fence_after_sync();
                const int64_t t = first + int64_t(c) * CT + r;
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    float y[32];
                    umma::tmem_ld32(tmem + T_O1 + 32 * i + lanes, y);
                    umma::tmem_wait_ld();
                    if (i == 1) {
                        umma::fence_before_sync();
                        arrive(o1_free);
                    }
                    if (t < p.T) {
                        __nv_bfloat16* const to = out + t * p.ot + 32 * i;
#pragma unroll
                        for (int e = 0; e < 32; e += 8) {
                            uint32_t w[4];
#pragma unroll
                            for (int k = 0; k < 4; ++k) w[k] = pack_bf16(x[i][e + 2 * k] + y[e + 2 * k], x[i][e + 2 * k + 1] + y[e + 2 * k + 1]);
                            if (col0 + 32 * i + e < p.dv) *reinterpret_cast<uint4*>(to + e) = make_uint4(w[0], w[1], w[2], w[3]);
                        }
                    }
                }
            }
        }
    } else if (warp == 12) {
        // ---------------------------------------------------------------- loads and MMAs
        if (lane == 0) {
            const int hq = h / p.q.share, hk = h / p.k.share, hv = h / p.v.share;
            int nq = 0, nk = 0, nv = 0;  // loads issued
            auto load_q = [&] {
                if (STATE || nq >= n) return;
                const int st = nq % NQ, t = static_cast<int>(first) + nq * CT;
                mbar_arrive_expect_tx(full_q + st, M::QB);
#pragma unroll
                for (int i = 0; i < DK / 64; ++i) tma_load(sb + M::Q + st * M::QB + i * CT * 128, &up.q, 64 * i, hq, t, b, full_q + st);
                ++nq;
            };
            auto load_k = [&] {
                if (nk >= n) return;
                const int st = nk % NK, t = static_cast<int>(first) + nk * CT;
                mbar_arrive_expect_tx(full_k + st, M::QB);
#pragma unroll
                for (int i = 0; i < DK / 64; ++i) tma_load(sb + M::K + st * M::QB + i * CT * 128, &up.k, 64 * i, hk, t, b, full_k + st);
                ++nk;
            };
            auto load_v = [&] {
                if (nv >= n) return;
                const int st = nv % NV, t = static_cast<int>(first) + nv * CT;
                mbar_arrive_expect_tx(full_v + st, M::VB);
                tma_load(sb + M::V + st * M::VB, &up.v, col0, hv, t, b, full_v + st);
                ++nv;
            };
            for (int i = 0; i < (NK > NQ ? NK : NQ); ++i) {
                if (i < NK) load_k();
                if (i < NQ) load_q();
                if (i < NV) load_v();
            }
            constexpr uint32_t ID_QK = umma::idesc_bf16(128, 128, umma::K_MAJOR, umma::K_MAJOR);
            constexpr uint32_t ID_QS = umma::idesc_bf16(128, DVS, umma::K_MAJOR, umma::K_MAJOR);
            constexpr uint32_t ID_PV = umma::idesc_bf16(128, DVS, umma::K_MAJOR, umma::MN_MAJOR);
            constexpr uint32_t ID_VK = umma::idesc_bf16(DVS, DK, umma::MN_MAJOR, umma::MN_MAJOR);
            auto issue_vk = [&](int c) {
                umma::fence_after_sync();
                const uint32_t k0 = sb + M::K + (c % NK) * M::QB;
#pragma unroll
                for (int a = kVPlanes - 1; a >= 0; --a)  // the smallest products first
#pragma unroll
                    for (int k = 0; k < CT / 16; ++k)
                        umma::mma_bf16(tmem + T_DS, umma::smem_desc(sb + M::W + a * M::VB + 2048 * k, CT * 128, 1024),
                                       umma::smem_desc(k0 + 2048 * k, CT * 128, 1024), ID_VK, a < kVPlanes - 1 || k > 0);
                umma::mma_commit(ds_done);
            };
            if constexpr (STATE) {
                for (int c = 0; c < n; ++c) {
                    wait(full_k + c % NK, c / NK);
                    wait(vw_ready, c);
                    if (c > 0) load_k(), load_v();  // chunk c - 1 has been read: its dS has been added
                    issue_vk(c);
                }
            } else {
                for (int c = 0; c <= n; ++c) {
                    if (c < n) {
                        wait(s_ready, c);
                        if (c > 0) load_k();  // chunk c - 1's MMAs with K are done: its dS has been added
                        wait(full_q + c % NQ, c / NQ);
                        wait(full_k + c % NK, c / NK);
                        if (c > 0) wait(o2_free, c - 1);
                        if (c > 1) wait(o_done, c - 2);  // P's buffer has been read
                        umma::fence_after_sync();
                        const uint32_t q0 = sb + M::Q + (c % NQ) * M::QB, k0 = sb + M::K + (c % NK) * M::QB;
#pragma unroll
                        for (int k = 0; k < DK / 16; ++k) {
                            const uint32_t off = (k >> 2) * (CT * 128) + 32 * (k & 3);
                            umma::mma_bf16(tmem + T_P + 128 * (c & 1), umma::smem_desc(q0 + off, 16, 1024),
                                           umma::smem_desc(k0 + off, 16, 1024), ID_QK, k > 0);
                        }
#pragma unroll
                        for (int a = 1; a >= 0; --a)
#pragma unroll
                            for (int k = 0; k < DK / 16; ++k)
                                umma::mma_bf16(tmem + T_O2, umma::smem_desc(q0 + (k >> 2) * (CT * 128) + 32 * (k & 3), 16, 1024),
                                               umma::smem_desc(sb + M::S + a * M::SB + (k >> 2) * (DVS * 128) + 32 * (k & 3), 16, 1024),
                                               ID_QS, a < 1 || k > 0);
                        umma::mma_commit(qk_done + (c & 1));
                    }
                    // whichever can go: dS of this chunk, O1 of the one before it, loads
                    bool vk = c < n, pv = c > 0, lq = c < n, lv = false;
                    for (uint32_t i = 0; vk || pv || lq || lv; ++i) {
                        if (vk && mbar_test_wait(vw_ready, c & 1)) issue_vk(c), vk = false;
                        if (lq && mbar_test_wait(qk_done + (c & 1), (c >> 1) & 1)) load_q(), lq = false;
                        if (pv && mbar_test_wait(p_ready + ((c - 1) & 1), ((c - 1) >> 1) & 1) &&
                            (c == 1 || mbar_test_wait(o1_free, (c - 2) & 1))) {
                            umma::fence_after_sync();
                            const uint32_t tp = tmem + T_P + 128 * ((c - 1) & 1), v0 = sb + M::V + ((c - 1) % NV) * M::VB;
#pragma unroll
                            for (int a = 1; a >= 0; --a)
#pragma unroll
                                for (int k = 0; k < CT / 16; ++k)
                                    mma_ts(tmem + T_O1, tp + 32 * (k >> 1) + 16 * a + 8 * (k & 1), umma::smem_desc(v0 + 2048 * k, CT * 128, 1024),
                                           ID_PV, a < 1 || k > 0);
                            umma::mma_commit(o_done);
                            pv = false, lv = true;
                        }
                        if (lv && mbar_test_wait(o_done, (c - 1) & 1)) load_v(), lv = false;
                        if (*dead) break;
                        if (i >= up.polls * 16) *dead = 1;
                    }
                }
            }
            // every MMA and load issued ends before the block does
            umma::mma_commit(drain);
            for (uint32_t i = 0; i < kPolls && !mbar_try_wait(drain, 0); ++i) {
            }
            auto landed = [&](uint64_t* full, int issued, int ring) {
                for (int l = issued > ring ? issued - ring : 0; l < issued; ++l)
                    for (uint32_t i = 0; i < kPolls && !mbar_try_wait(full + l % ring, (l / ring) & 1); ++i) {
                    }
            };
            landed(full_q, nq, NQ), landed(full_k, nk, NK), landed(full_v, nv, NV);
        }
        __syncwarp();
    } else {
        // ---------------------------------------------------------------- decays
        Tokens next = load_tokens(p, ld, marks, first);
        for (int c = 0; c < n; ++c) {
            const Tokens now = next;
            if (c + 1 < n) next = load_tokens(p, ld, marks, first + int64_t(c + 1) * CT);
            if (c >= GR) wait(gates_free + c % GR, c / GR - 1);
            make_gates(now, p.scale, gates[c % GR]);
            arrive(gates_full + c % GR);
        }
    }
    umma::fence_before_sync();
    __syncthreads();
    if (warp == 12) {
        umma::fence_after_sync();
        umma::tmem_dealloc(tmem, kTmem);
    }
    if (threadIdx.x == 0) up.redo[blockIdx.x] = *dead || *bad_word ? 1u : 0u;
}

// ------------------------------------------------------------------ host
// [nb, T, heads, features], features next to each other, as boxes of 128 tokens x 64.
int encode(CUtensorMap* tm, const Stream& x, int64_t nb, int64_t T, int64_t heads, int64_t features) {
    const int64_t any = (features * 2 + 15) / 16 * 16;  // a stride that no step is taken with
    const cuuint64_t dims[4] = {cuuint64_t(features), cuuint64_t(heads), cuuint64_t(T), cuuint64_t(nb)};
    const cuuint64_t gs[3] = {cuuint64_t(heads > 1 ? x.sh * 2 : any), cuuint64_t(T > 1 ? x.st * 2 : any), cuuint64_t(nb > 1 ? x.sb * 2 : any)};
    const cuuint32_t box[4] = {64, 1, CT, 1}, es[4] = {1, 1, 1, 1};
    auto fn = encode_fn();
    if (fn == nullptr) return fail(NEED_ERR_CUDA, "cuTensorMapEncodeTiled entry point unavailable");
    const CUresult r = fn(tm, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(x.p), dims, gs, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
                          CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? NEED_OK : fail(NEED_ERR_CUDA, "cuTensorMapEncodeTiled failed: %d", int(r));
}

std::atomic<uint32_t> umma_polls{kPolls};

template <int DK, bool STATE>
int launch(const UmmaParams& up, int64_t blocks, cudaStream_t s) {
    static std::atomic<uint64_t> done{0};
    auto kern = umma_attention_kernel<DK, STATE>;
    cudaError_t e = ensure_smem(kern, Map<DK>::BYTES, done);
    if (e != cudaSuccess) return cuda_fail(e, "linear attention shared memory");
    kern<<<static_cast<unsigned>(blocks), kThreads, Map<DK>::BYTES, s>>>(up);
    e = cudaGetLastError();
    return e == cudaSuccess ? NEED_OK : cuda_fail(e, "linear attention launch");
}

}  // namespace

namespace need {
namespace attention {

// bf16 with rows of whole, aligned 16-byte pieces (the caller has seen to that): what a tensor
// map can say of the strides.
bool umma_takes(const AttnParams& p, int64_t nb) {
    auto in = [](int64_t n, int64_t stride) { return n <= 1 || (stride > 0 && stride < (int64_t(1) << 38)); };
    for (const Stream* x : {&p.q, &p.k, &p.v})
        if (!in(p.H / x->share, x->sh) || !in(p.T, x->st) || !in(nb, x->sb)) return false;
    return p.T < (int64_t(1) << 31) - 256 && nb < (int64_t(1) << 31) && p.ob % 8 == 0 && p.ot % 8 == 0 && p.oh % 8 == 0;
}

int umma_run(const AttnParams& p, int64_t nb, bool state, uint32_t* redo, cudaStream_t stream) {
    if (int rc = ensure_context()) return rc;
    UmmaParams up{};
    up.a = p, up.redo = redo, up.polls = umma_polls.load(std::memory_order_relaxed);
    if (int rc = encode(&up.q, p.q, nb, p.T, p.H / p.q.share, p.dk)) return rc;
    if (int rc = encode(&up.k, p.k, nb, p.T, p.H / p.k.share, p.dk)) return rc;
    if (int rc = encode(&up.v, p.v, nb, p.T, p.H / p.v.share, p.dv)) return rc;
    const int64_t blocks = nb * p.H * p.slices * (state ? p.nseg - 1 : p.nseg);
    if (p.dk <= 64) return state ? launch<64, true>(up, blocks, stream) : launch<64, false>(up, blocks, stream);
    return state ? launch<128, true>(up, blocks, stream) : launch<128, false>(up, blocks, stream);
}

}  // namespace attention
}  // namespace need

extern "C" void need_test_linear_attention_polls(uint32_t polls) { umma_polls.store(polls == 0 ? kPolls : polls, std::memory_order_relaxed); }
