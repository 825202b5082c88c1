// linear_attention_umma.cu -- linear attention with a decay for each head on sm_100a's
// tensor cores (tcgen05): bf16, up to 128 features, rows of whole 16 bytes.  The
// mathematics, the planes and the segments are those of linear_attention.cu; the
// chunks have 128 tokens.
//
// One CTA walks the chunks of one (sequence, head, 64 columns of v).  Per chunk, with
// fp32 accumulators in tensor memory:
//
//   P    = Q K^T                 128 x 128
//   O2   = Q S                   128 x 64           S: 2 planes, shared memory; two buffers
//   O1   = P' V                  128 x 64           P' = P with its decays, 2 planes, in P's place; two buffers at
//                                                   128 features, where P has one
//   dS^T = (V w)^T K             64 x features      V w: 3 planes, shared memory
//   out  = O1 + e^G O2,  S' = e^{G_end} S + dS
//
// The state lies in the registers of the warps that add dS to it.  Each kind of work has
// warps of its own, which meet at mbarriers only, so that a chunk's scores, outputs and
// state run beside its neighbours':
//
//   warps 0-7    P' and the outputs: two for each 32 rows, a row per thread.  A decay is a row's
//                factor, which can wait for the outputs, times a column's -- but in a chunk that a
//                segment starts in, or that decays by more than 2^-64 or grows by more than 2^32
//   warps 8-15   V w, the check for infinities, the state and its planes
//   warp 16      the decays of the chunks ahead
//   warps 17-19  the MMAs, each with the loads (TMA, no multicast) whose place they free: P and
//                O2; dS; O1.  One elected lane issues.
//
// All roles' code runs on every part of the multiprocessor, so that it is kept short: straight
// code of the same work took twice the time, waiting for instructions.
//
// Every wait is bounded.  A block that gave one up, or has an output or a state that is not finite (or
// a log decay that makes a chunk's products leave fp32's range), says so in `redo`:
// attention_kernel, launched behind, then computes the block's whole segment.
//
// Measured: 16 x 4096 tokens, 16 heads of 64 x 64, 161 us (3.4 TB/s of the 541 MB that go in
// and out; attention_kernel 390); 8 x 2048, 13 heads of 64 x 64, 44 us (104 chains leave 44 of
// the 148 multiprocessors idle); 1 x 16384, 32 heads of 128 x 128, 254-264 us, in three segments
// of each chain, the middle one run twice.  A chunk takes 2.0 us at 64 features (the MMAs 1.1, the
// warps' work on P', outputs and state beside them about the whole) and 2.9 at 128 (the
// MMAs 1.9; one buffer of Q fits, which the products with K and S must have left before
// the next chunk's 32 KB come, and those take a third of the time).
#include <cuda.h>
#include <cuda_bf16.h>

#include <algorithm>
#include <type_traits>

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
constexpr int kThreads = 640;
constexpr int GR = 4;        // chunks whose decays are held
constexpr uint32_t kPolls = 1u << 16;  // of a wait before it is given up
constexpr uint32_t kTmem = 512, T_O1 = 0;  // tensor memory columns

struct alignas(16) Gates {
    float hi[CT], lo[CT], w[CT], eg[CT];  // as Decays
    float row[CT];  // what a row of O1 is multiplied with: where a decay is a row's factor times a column's
                    // (w), scale times that from the chunk's end back to the token; else 1
    int seg[CT];
    float d;
    int wild, factors;
};

// VP: planes of V w.  3 where the state itself is a result; where only outputs of bf16 come
// of it, 2 as of the other operands (16x4096 16x64 157 us, 165 with 3, when it was chosen).
template <int DK>
struct Map {  // shared memory, from a 1024-byte aligned base
    static constexpr int NQ = DK == 64 ? 2 : 1, NK = DK == 64 ? 3 : 2, NV = NK;  // chunks loaded ahead
    // buffers of P (tensor memory holds a second one at 64 features; at 128 in the place of O2's
    // second, which took longer: 1x16384 32x128 406 us against 343)
    static constexpr int NP = DK == 64 ? 2 : 1, NO = 3 - NP;  // NO: of O1
    static constexpr uint32_t T_O2 = T_O1 + NO * DVS, T_DS = T_O2 + 2 * DVS, T_P = T_DS + DK;
    static_assert(T_P + NP * 128 <= kTmem, "tensor memory");
    static constexpr int QB = CT * DK * 2, VB = CT * DVS * 2, SB = DVS * DK * 2;
    static constexpr int Q = 0, K = Q + NQ * QB, V = K + NK * QB, W = V + NV * VB, S = W + 3 * VB, G = S + 2 * SB;
    static constexpr int BAR = G + GR * static_cast<int>(sizeof(Gates)), BYTES = BAR + 512 + 1024;
};

struct UmmaParams {
    CUtensorMap q, k, v;  // [sequence, token, head, feature], boxes of 128 tokens x 64 features
    AttnParams a;
    uint32_t* redo;
    uint32_t polls;
    int32_t wide;  // the outputs' rows lie apart by whole 32 bytes
};

__device__ __forceinline__ void tma_load(uint32_t dst, const CUtensorMap* tm, int c0, int c1, int c2, int c3, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst), "l"(tm), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(bar)
        : "memory");
}
__device__ __forceinline__ void st_shared(uint32_t to, uint32_t v) { asm volatile("st.shared.b32 [%0], %1;" ::"r"(to), "r"(v) : "memory"); }
__device__ __forceinline__ bool try_wait(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(bar), "r"(parity)
        : "memory");
    return ok != 0;
}
// Bounded; after one wait was given up (the word at `dead`) nobody waits any more.
__device__ __noinline__ void wait_on(uint32_t bar, uint32_t parity, uint32_t dead, uint32_t polls) {
    for (uint32_t i = 1; !try_wait(bar, parity); ++i) {
        if (i % 64 != 0 && i < polls) continue;
        uint32_t d;
        asm volatile("ld.volatile.shared.u32 %0, [%1];" : "=r"(d) : "r"(dead) : "memory");
        if (d != 0) return;
        if (i >= polls) asm volatile("st.volatile.shared.u32 [%0], %1;" ::"r"(dead), "r"(1u) : "memory");
    }
}
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
    return p != 0;
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
// 16 words into this thread's lane
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&v)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
        "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]),
        "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
        : "memory");
}
// 16 fp32 columns of this thread's lane
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, float (&v)[16]) {
    uint32_t r[16];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
          "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr));
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r[i]);
}
// 32 or 64 columns of 16 lanes: the four values of 8 columns lie as in a 16 x 8 accumulator
// of mma.sync (rows lane / 4 and + 8, columns 2 (lane % 4) and + 1).
__device__ __forceinline__ void tmem_ld_half(uint32_t taddr, float (&v)[16]) {
    uint32_t r[16];
    asm volatile(
        "tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
          "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr));
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r[i]);
}

// ------------------------------------------------------------------ decays
// A sum as two floats: a + b with what rounding left of it (Knuth's two-sum).
struct Sum2 {
    float hi, lo;
};
__device__ __forceinline__ Sum2 add(const Sum2& a, const Sum2& b) {
    const float s = a.hi + b.hi, t = s - a.hi;
    return {s, ((a.hi - (s - t)) + (b.hi - t)) + (a.lo + b.lo)};
}
__device__ __forceinline__ float minus(const Sum2& a, const Sum2& b) { return (a.hi - b.hi) + (a.lo - b.lo); }

// One warp; x, the lane's 4 log decays (tokens 4 lane + e), -infinity where a segment starts.
// The running sums hold some 44 bits: sums of fp64 took three times the time.
__device__ __forceinline__ void make_gates(const float (&x)[4], float scale, Gates& g) {
    const int lane = threadIdx.x & 31;
    Sum2 G[4], sum{0.0f, 0.0f};
    int s = 0, send = 0;
    bool wild = false, reset[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        reset[e] = x[e] == -INFINITY;
        wild |= !(x[e] <= 0.5f);  // 128 of them stay below 2^93
        // a token's state falls below every fp32 value long before e^-10000; a NaN stays one
        const float v = reset[e] ? 0.0f : x[e] < -10000.0f ? -10000.0f : x[e];
        constexpr float l2e = 1.4426950408889634f, l2e_lo = 1.9259629911266175e-8f;  // log2(e) as two floats
        const float y = v * l2e;
        sum = add(sum, {y, fmaf(v, l2e, -y) + v * l2e_lo});
        G[e] = sum;
        const uint32_t m = __ballot_sync(0xffffffffu, reset[e]);
        s += __popc(m & ((1u << lane) - 1u)), send += __popc(m);
    }
    Sum2 incl = sum;
#pragma unroll
    for (int m = 1; m < 32; m <<= 1) {
        const Sum2 o{__shfl_up_sync(0xffffffffu, incl.hi, m), __shfl_up_sync(0xffffffffu, incl.lo, m)};
        if (lane >= m) incl = add(o, incl);
    }
    auto of = [&](int l) { return Sum2{__shfl_sync(0xffffffffu, incl.hi, l), __shfl_sync(0xffffffffu, incl.lo, l)}; };
    Sum2 before = of((lane + 31) & 31);
    if (lane == 0) before = {0.0f, 0.0f};
    const Sum2 end = of(31);
    // a row's factor is up to 2^64 then, a column's up to 2^32 (more than 1 only where states grow), and
    // neither falls below what bf16 holds
    bool near = send == 0 && end.hi > -64.0f;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        G[e] = add(before, G[e]);
        const float d = minus(G[e], end);
        near = near && d < 64.0f && d > -32.0f;
    }
    const bool factors = __all_sync(0xffffffffu, near);
    float4 hi, lo, w, eg, be;
    int4 seg;
    float *ph = &hi.x, *pl = &lo.x, *pw = &w.x, *pe = &eg.x, *pb = &be.x;
    int* ps = &seg.x;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const Sum2 t = G[e];
        s += reset[e] ? 1 : 0;
        ph[e] = t.hi, pl[e] = t.lo, ps[e] = s;
        pw[e] = s == send ? ex2(minus(end, t)) : 0.0f;
        pe[e] = s == 0 ? scale * ex2(t.hi + t.lo) : 0.0f;
        pb[e] = factors ? scale * ex2(minus(t, end)) : 1.0f;
    }
    reinterpret_cast<float4*>(g.hi)[lane] = hi, reinterpret_cast<float4*>(g.lo)[lane] = lo, reinterpret_cast<float4*>(g.w)[lane] = w;
    reinterpret_cast<float4*>(g.eg)[lane] = eg, reinterpret_cast<float4*>(g.row)[lane] = be, reinterpret_cast<int4*>(g.seg)[lane] = seg;
    wild = __any_sync(0xffffffffu, wild);
    if (lane == 0) g.d = send == 0 ? ex2(end.hi + end.lo) : -1.0f, g.wild = wild ? 1 : 0, g.factors = factors ? 1 : 0;
}

// One lane of a warp: a chunk's 128 rows of one tensor, 64 columns at a time.
__device__ __noinline__ void load_rows(uint32_t full, const CUtensorMap* tm, uint32_t to, int bytes, int col, int head, int t, int b) {
    if (elect_one()) {
        asm volatile("mbarrier.arrive.expect_tx.release.cta.shared::cta.b64 _, [%0], %1;" ::"r"(full), "r"(bytes) : "memory");
#pragma unroll 1
        for (int j = 0; j < bytes; j += CT * 128) tma_load(to + j, tm, col + j / 256, head, t, b, full);
    }
    __syncwarp();
}

// The same rows into L2.
__device__ __forceinline__ void prefetch_rows(const CUtensorMap* tm, int bytes, int head, int t, int b) {
    if (elect_one())
#pragma unroll 1
        for (int j = 0; j < bytes; j += CT * 128)
            asm volatile("cp.async.bulk.prefetch.tensor.4d.L2.global.tile [%0, {%1, %2, %3, %4}];" ::"l"(tm), "r"(j / 256), "r"(head), "r"(t), "r"(b)
                         : "memory");
    __syncwarp();
}

// ------------------------------------------------------------------ the kernel
template <int DK, int VP>
__global__ void __launch_bounds__(kThreads, 1) umma_attention_kernel(const __grid_constant__ UmmaParams up) {
    using M = Map<DK>;
    constexpr int NQ = M::NQ, NK = M::NK, NV = M::NV, NP = M::NP;
    const AttnParams& p = up.a;
    extern __shared__ unsigned char smem_raw[];
    unsigned char* const base = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const uint32_t sb = smem_addr(base);
    uint64_t* bar = reinterpret_cast<uint64_t*>(base + M::BAR);
    // Those with two by turns are told apart so that none is asked of a phase that another has
    // followed: a waiter may be a chunk behind.
    uint64_t *full_q = bar, *full_k = full_q + NQ, *full_v = full_k + NK, *gates_full = full_v + NV, *gates_free = gates_full + GR,
             *k_free = gates_free + GR, *v_free = k_free + NK, *s_ready = v_free + NV, *vw_ready = s_ready + 1,
             *qk_done = vw_ready + 1 /* 2 */, *qs_done = qk_done + 2 /* 2 */, *ds_done = qs_done + 2, *ds_free = ds_done + 1,
             *p_ready = ds_free + 1 /* 2 */, *o_done = p_ready + 2 /* 2 */, *o_free = o_done + 2 /* 2 */, *drain = o_free + 2 /* 3 */;
    uint32_t* const tbase = reinterpret_cast<uint32_t*>(drain + 3);
    volatile uint32_t* const dead = tbase + 1;
    uint32_t* const bad_word = tbase + 2;
    Gates* const gates = reinterpret_cast<Gates*>(base + M::G);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t segs = p.launched(), rest = blockIdx.x / segs;
    const int seg = static_cast<int>(blockIdx.x % segs) + (p.ahead ? 0 : p.lead), slice = static_cast<int>(rest % p.slices);
    const bool state = p.ahead && seg >= p.lead;  // only the state
    const int64_t chain = rest / p.slices;
    const int b = static_cast<int>(static_cast<uint32_t>(chain) / p.H), h = static_cast<int>(static_cast<uint32_t>(chain) % p.H), col0 = slice * DVS;
    const int64_t first = p.segment(seg) * 64, last = p.segment(seg + 1) * 64 < p.T ? p.segment(seg + 1) * 64 : p.T;
    const int n = static_cast<int>((last - first + CT - 1) / CT);
    const float* ld = p.ld + b * p.lb + h * p.lh;
    const uint8_t* marks = p.seg == nullptr ? nullptr : p.seg + b * p.gb;

    if (threadIdx.x == 0) {
        auto init = [](uint64_t* x, int n, int count) {  // arrivals: of warps, or of MMAs and loads
#pragma unroll 1
            for (int i = 0; i < n; ++i) mbar_init(x + i, count);
        };
        init(full_q, NQ + NK + NV + GR, 1), init(gates_free, GR, state ? 8 : 16), init(k_free, NK, state ? 1 : 2);
        init(v_free, NV, state ? 8 : 9), init(s_ready, 2, 8), init(qk_done, 5, 1), init(ds_free, 1, 8), init(p_ready, 2, 8);
        init(o_done, 2, 1), init(o_free, 2, 8), init(drain, 3, 1);
        *dead = 0, *bad_word = 0;
        fence_barrier_init();
    }
    if (warp == 16) {
        umma::tmem_alloc(tbase, kTmem);
        umma::tmem_relinquish();
    }
    umma::fence_before_sync();
    __syncthreads();
    umma::fence_after_sync();
    const uint32_t tmem = *tbase;
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;  // this warp's part of tensor memory

    auto wait = [&](const uint64_t* x, uint32_t phase) {
        const uint32_t at = smem_addr(x);
        if (!try_wait(at, phase & 1u)) wait_on(at, phase & 1u, smem_addr(tbase + 1), up.polls);
    };
    auto arrive = [&](uint64_t* x) {  // one of a warp's lanes, for all
        __syncwarp();
        if (lane == 0) mbar_arrive(x);
    };

    if (warp < 8) {
        // ---------------------------------------------------------------- P', outputs
        if (!state) {
            const int quad = warp & 3, half = warp >> 2, r = 32 * quad + lane;
            __nv_bfloat16* const out = static_cast<__nv_bfloat16*>(p.out) + b * p.ob + h * p.oh + col0 + 32 * half;
            const int cols = p.dv - col0 - 32 * half;
            float eg_last = 0.0f, row_last = 0.0f;  // of the chunk whose outputs come next
            bool reach_last = false;                // whether the entering state reaches its row
            float2 chk = splat(0.0f);               // 0 unless an output is no finite number
            auto outputs = [&](int c) {  // 32 columns of chunk c
                wait(o_done + (c & 1), c >> 1);
                wait(qs_done + (c & 1), c >> 1);
                umma::fence_after_sync();
                float x[32], y[32];
                umma::tmem_ld32(tmem + T_O1 + DVS * (c % M::NO) + 32 * half + lanes, x);
                umma::tmem_ld32(tmem + M::T_O2 + DVS * (c & 1) + 32 * half + lanes, y);
                umma::tmem_wait_ld();
                umma::fence_before_sync();
                arrive(o_free + (c & 1));
                const int64_t t = first + int64_t(c) * CT + r;
                __nv_bfloat16* const to = out + t * p.ot;
#pragma unroll
                for (int e = 0; e < 32; e += 16) {
                    uint32_t w[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        float2 z = __fmul2_rn(splat(row_last), make_float2(x[e + 2 * i], x[e + 2 * i + 1]));
                        if (reach_last) z = __ffma2_rn(splat(eg_last), make_float2(y[e + 2 * i], y[e + 2 * i + 1]), z);
                        chk = __ffma2_rn(z, splat(0.0f), chk);
                        w[i] = pack_bf16(z.x, z.y);
                    }
                    if (t >= p.T) continue;
                    if (up.wide && e + 16 <= cols) {
                        asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(to + e), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]),
                                     "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
                                     : "memory");
                    } else {
                        if (e < cols) *reinterpret_cast<uint4*>(to + e) = make_uint4(w[0], w[1], w[2], w[3]);
                        if (e + 8 < cols) *reinterpret_cast<uint4*>(to + e + 8) = make_uint4(w[4], w[5], w[6], w[7]);
                    }
                }
            };
#pragma unroll 1
            for (int c = 0; c <= n; ++c) {  // P' of chunk c, the outputs of the one before it
                float eg = 0.0f, row = 0.0f;  // of the chunk
                bool reach = false;
                if (c < n) {
                    const Gates& g = gates[c % GR];
                    wait(gates_full + c % GR, c / GR);
                    eg = g.eg[r], row = g.row[r], reach = g.seg[r] == 0;
                    const bool factors = g.factors != 0;
                    wait(qk_done + (c & 1), c >> 1);
                    umma::fence_after_sync();
                    const uint32_t tp = tmem + M::T_P + 128 * (c % NP) + lanes;
                    // 16 columns at a time, every other one, two of them in flight; after the diagonal's they are 0
                    auto scores = [&](int cb, float (&x)[16]) {
                        uint32_t pl[16];  // the first planes of 16 scores, then the second
                        if (cb < 2 * quad + 2) {
                            if (factors) {
#pragma unroll
                                for (int e = 0; e < 16; e += 4) {
                                    const float4 w = *reinterpret_cast<const float4*>(&g.w[16 * cb + e]);
                                    const float2 u = __fmul2_rn(make_float2(x[e], x[e + 1]), make_float2(w.x, w.y));
                                    const float2 d = __fmul2_rn(make_float2(x[e + 2], x[e + 3]), make_float2(w.z, w.w));
                                    x[e] = u.x, x[e + 1] = u.y, x[e + 2] = d.x, x[e + 3] = d.y;
                                }
                                if (cb >= 2 * quad)
#pragma unroll
                                    for (int e = 0; e < 16; ++e) x[e] = 16 * cb + e <= r ? x[e] : 0.0f;
                            } else {
                                const float hr = g.hi[r], lr = g.lo[r];
                                const int sr = g.seg[r];
#pragma unroll
                                for (int e = 0; e < 16; ++e) {
                                    const int i = 16 * cb + e;
                                    x[e] = g.seg[i] == sr && i <= r ? x[e] * (p.scale * ex2((hr - g.hi[i]) + (lr - g.lo[i]))) : 0.0f;
                                }
                            }
#pragma unroll
                            for (int e = 0; e < 8; ++e) {
                                uint32_t two[2];
                                split<2>(make_float2(x[2 * e], x[2 * e + 1]), two);
                                pl[e] = two[0], pl[8 + e] = two[1];
                            }
                        } else {
#pragma unroll
                            for (int e = 0; e < 16; ++e) pl[e] = 0u;
                        }
                        tmem_st16(tp + 16 * cb, pl);
                    };
#pragma unroll 1
                    for (int cb = half; cb < 8; cb += 4) {
                        float x[16], y[16];
                        tmem_ld16(tp + 16 * cb, x);
                        tmem_ld16(tp + 16 * cb + 32, y);
                        umma::tmem_wait_ld();
                        scores(cb, x);
                        scores(cb + 2, y);
                    }
                    umma::tmem_wait_st();
                    umma::fence_before_sync();
                    arrive(p_ready + (c & 1));
                    arrive(gates_free + c % GR);
                }
                if (c > 0) outputs(c - 1);
                eg_last = eg, row_last = row, reach_last = reach;
            }
            if (!(chk.x == 0.0f && chk.y == 0.0f)) *bad_word = 1;
        }
    } else if (warp < 16) {
        // ---------------------------------------------------------------- V w, the state
        // 16 columns of v and half of the features a warp
        constexpr int NH = DK / 16;  // 8-feature tiles of a warp
        const int bt = threadIdx.x - 256, quad = warp & 3, gr = lane >> 2, c2 = (lane & 3) * 2, j0 = col0 + 16 * quad + gr;
        const int m0 = (warp >= 12 ? NH : 0);  // its first tile
        float s[NH][4];  // transposed: rows j0 and + 8, columns 8 (m0 + m) + c2 and + 1
        {
            const float* from = state ? nullptr : seg > 0 ? p.part + (chain * (p.nseg - 1) + seg - 1) * p.dk * int64_t(p.dv)
                                      : p.s0 != nullptr   ? p.s0 + chain * p.dk * int64_t(p.dv) : nullptr;
            if (from != nullptr && starts(ld, p.lt, marks, p.gt, first)) from = nullptr;  // nothing of it is seen
#pragma unroll
            for (int m = 0; m < NH; ++m)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int i = 8 * (m0 + m) + c2 + (e & 1), j = j0 + (e >> 1) * 8;
                    s[m][e] = from != nullptr && i < p.dk && j < p.dv ? from[int64_t(i) * p.dv + j] : 0.0f;
                }
            if (from != nullptr) {
                float chk = 0.0f;
#pragma unroll
                for (int m = 0; m < NH; ++m)
#pragma unroll
                    for (int e = 0; e < 4; ++e) chk = fmaf(s[m][e], 0.0f, chk);
                if (!(chk == 0.0f)) *bad_word = 1;
            }
        }
        float d, d_next = 0.0f;
        bool bad = false;
        float2 vw[16];  // of the next chunk, 4 rows 32 apart: made while its predecessor's dS is
        auto fetch = [&](int c) {
            const Gates& g = gates[c % GR];
            wait(full_v + c % NV, c / NV);
            wait(gates_full + c % GR, c / GR);
            const unsigned char* vt = base + M::V + (c % NV) * M::VB + umma::sw128(bt / 8, bt % 8);  // rows 32 apart: 4096 bytes
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint4 u = *reinterpret_cast<const uint4*>(vt + 4096 * i);
                const float2 w = splat(g.w[bt / 8 + 32 * i]);
                vw[4 * i] = __fmul2_rn(w, unpack_bf16(u.x)), vw[4 * i + 1] = __fmul2_rn(w, unpack_bf16(u.y));
                vw[4 * i + 2] = __fmul2_rn(w, unpack_bf16(u.z)), vw[4 * i + 3] = __fmul2_rn(w, unpack_bf16(u.w));
            }
            d_next = g.d;
            bad |= g.wild != 0;
            arrive(gates_free + c % GR);
            arrive(v_free + c % NV);
        };
        fetch(0);
        for (int c = 0; c < n; ++c) {
            // (the planes of the last chunk have been read: its dS is there)
            unsigned char* const wt = base + M::W + umma::sw128(bt / 8, bt % 8);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                uint32_t pl[4][VP];
#pragma unroll
                for (int e = 0; e < 4; ++e) split<VP>(vw[4 * i + e], pl[e]);
#pragma unroll
                for (int a = 0; a < VP; ++a)
                    *reinterpret_cast<uint4*>(wt + a * M::VB + 4096 * i) = make_uint4(pl[0][a], pl[1][a], pl[2][a], pl[3][a]);
            }
            fence_proxy_async_shared();
            arrive(vw_ready);
            d = d_next;
            if (!state) {  // the planes of the state that enters, as the K-major B of Q S
                if (c > 0) wait(qs_done + ((c - 1) & 1), (c - 1) >> 1);  // the last ones have been read
                const uint32_t row = sb + M::S + umma::sw128(16 * quad + gr, 0) + c2 * 2;  // and the one 8 below, 1024 bytes on
#pragma unroll
                for (int m = 0; m < NH; ++m) {
                    // the row's 16-byte piece k lies at k ^ gr, piece 0 at gr
                    const uint32_t to = (row ^ (((m0 + m) & 7) << 4)) + ((m0 + m) >> 3) * (DVS * 128);
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        uint32_t two[2];
                        split<2>(make_float2(s[m][2 * r], s[m][2 * r + 1]), two);
                        st_shared(to + r * 1024, two[0]), st_shared(to + r * 1024 + M::SB, two[1]);
                    }
                }
                fence_proxy_async_shared();
                arrive(s_ready);
            }
            if (c + 1 < n) fetch(c + 1);
            wait(ds_done, c);
            umma::fence_after_sync();
            // an infinity or NaN of k, v or the state leaves one here, under a weight of 0 too (V w is a
            // NaN then): a sum of 0 x is 0 otherwise
            float2 chk = splat(0.0f);
            const float2 dd = splat(d == -1.0f ? 0.0f : d);
#pragma unroll
            for (int m1 = 0; m1 < NH; m1 += 4) {
                float x[16];
                tmem_ld_half(tmem + M::T_DS + 8 * (m0 + m1) + lanes, x);
                umma::tmem_wait_ld();
                if (m1 + 4 == NH) {
                    umma::fence_before_sync();
                    arrive(ds_free);
                }
#pragma unroll
                for (int m = 0; m < 4; ++m)
#pragma unroll
                    for (int e = 0; e < 4; e += 2) {
                        const float2 z = make_float2(x[4 * m + e], x[4 * m + e + 1]);
                        float2 y = make_float2(s[m1 + m][e], s[m1 + m][e + 1]);
                        if (d == -1.0f) y = splat(0.0f);  // whatever it holds
                        y = __ffma2_rn(dd, y, z);
                        chk = __ffma2_rn(y, splat(0.0f), chk);
                        s[m1 + m][e] = y.x, s[m1 + m][e + 1] = y.y;
                    }
            }
            bad |= !(chk.x == 0.0f && chk.y == 0.0f);
        }
        if (bad) *bad_word = 1;
        float* const to = p.ahead ? p.part + (chain * (p.nseg - 1) + seg) * p.dk * int64_t(p.dv)
                                : seg == p.nseg - 1 && p.sT != nullptr ? p.sT + chain * p.dk * int64_t(p.dv) : nullptr;
        if (to != nullptr)
#pragma unroll
            for (int m = 0; m < NH; ++m)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int i = 8 * (m0 + m) + c2 + (e & 1), j = j0 + (e >> 1) * 8;
                    if (i < p.dk && j < p.dv) to[int64_t(i) * p.dv + j] = s[m][e];
                }
    } else if (warp == 16) {
        // ---------------------------------------------------------------- decays
        const float* at = ld + (first + 4 * lane) * p.lt;
        const uint8_t* mark = marks == nullptr ? nullptr : marks + (first + 4 * lane) * p.gt;
        float next[4];
        auto fetch = [&](int c) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const bool live = first + c * CT + 4 * lane + i < p.T;
                next[i] = live ? at[i * p.lt] : 0.0f;
                if (live && marks != nullptr && mark[i * p.gt] != 0) next[i] = -INFINITY;
            }
            at += CT * p.lt;
            if (marks != nullptr) mark += CT * p.gt;
        };
        fetch(0);
        double* const total = reinterpret_cast<double*>(base + M::BAR + 504);  // the segment's decay, lane 0's: no registers for it
        if (lane == 0) *total = 1.0;
#pragma unroll 1
        for (int c = 0; c < n; ++c) {
            float now[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) now[i] = next[i];
            if (c + 1 < n) fetch(c + 1);
            if (c >= GR) wait(gates_free + c % GR, c / GR - 1);
            make_gates(now, p.scale, gates[c % GR]);
            if (p.ahead && lane == 0) *total = *total == -1.0 || gates[c % GR].d == -1.0f ? -1.0 : *total * gates[c % GR].d;
            arrive(gates_full + c % GR);
        }
        if (p.ahead && slice == 0 && lane == 0) put_decay(p.part_d + 2 * (chain * (p.nseg - 1) + seg), *total);
    } else {
        // ---------------------------------------------------------------- MMAs and loads
        const uint64_t desc_k = umma::smem_desc(sb, 16, 1024), desc_mn = umma::smem_desc(sb, CT * 128, 1024);  // + bytes / 16
        auto load = [&](uint64_t* full, const CUtensorMap* tm, uint32_t to, int bytes, int col, int head, int c) {
            if (c < n) load_rows(smem_addr(full), tm, to, bytes, col, head, static_cast<int>(first) + c * CT, b);
        };
        auto load_q = [&](int c) { load(full_q + c % NQ, &up.q, sb + M::Q + c % NQ * M::QB, M::QB, 0, h / p.q.share, c); };
        auto load_k = [&](int c) { load(full_k + c % NK, &up.k, sb + M::K + c % NK * M::QB, M::QB, 0, h / p.k.share, c); };
        auto load_v = [&](int c) { load(full_v + c % NV, &up.v, sb + M::V + c % NV * M::VB, M::VB, col0, h / p.v.share, c); };
        if (warp == 17) {  // P = Q K^T of the chunk ahead, O2 = Q S
            if (!state) {
                constexpr uint32_t ID_QK = umma::idesc_bf16(128, 128, umma::K_MAJOR, umma::K_MAJOR);
                constexpr uint32_t ID_QS = umma::idesc_bf16(128, DVS, umma::K_MAJOR, umma::K_MAJOR);
#pragma unroll 1
                for (int c = 0; c < NQ; ++c) load_q(c);
                for (int c = 0; c <= n; ++c) {  // P of chunk c, O2 of the one before it
                    auto scores = [&] {
                        wait(full_q + c % NQ, c / NQ);
                        wait(full_k + c % NK, c / NK);
                        if (c >= NP) wait(o_done + ((c - NP) & 1), (c - NP) >> 1);  // the scores in P's place have been read
                        umma::fence_after_sync();
                        if (elect_one()) {
                            const uint64_t q0 = desc_k + ((M::Q + (c % NQ) * M::QB) >> 4), k0 = desc_k + ((M::K + (c % NK) * M::QB) >> 4);
#pragma unroll 4
                            for (int k = 0; k < DK / 16; ++k) {
                                const uint32_t off = ((k >> 2) * (CT * 128) + 32 * (k & 3)) >> 4;
                                umma::mma_bf16(tmem + M::T_P + 128 * (c % NP), q0 + off, k0 + off, ID_QK, k > 0);
                            }
                            umma::mma_commit(qk_done + (c & 1));
                            umma::mma_commit(k_free + c % NK);
                        }
                        __syncwarp();
                    };
                    if (NQ > 1 && c < n) scores();
                    if (c > 0) {
                        const int l = c - 1;
                        wait(s_ready, l);
                        if (l > 1) wait(o_free + (l & 1), (l - 2) >> 1);  // the outputs two chunks back are read
                        umma::fence_after_sync();
                        if (elect_one()) {
                            const uint64_t q0 = desc_k + ((M::Q + (l % NQ) * M::QB) >> 4), s0 = desc_k + (M::S >> 4);
#pragma unroll 1
                            for (int a = 1; a >= 0; --a)
#pragma unroll 4
                                for (int k = 0; k < DK / 16; ++k)
                                    umma::mma_bf16(tmem + M::T_O2 + DVS * (l & 1), q0 + (((k >> 2) * (CT * 128) + 32 * (k & 3)) >> 4),
                                                   s0 + ((a * M::SB + (k >> 2) * (DVS * 128) + 32 * (k & 3)) >> 4), ID_QS, a < 1 || k > 0);
                            umma::mma_commit(qs_done + (l & 1));
                        }
                        __syncwarp();
                        if (l + NQ < n) {
                            wait(qs_done + (l & 1), l >> 1);  // and the scores before it
                            load_q(l + NQ);
                        }
                    }
                    if (NQ == 1 && c + 1 < n) prefetch_rows(&up.q, M::QB, h / p.q.share, static_cast<int>(first) + (c + 1) * CT, b);
                    if (NQ == 1 && c < n) scores();
                }
            }
        } else if (warp == 18) {  // dS = (V w)^T K
            constexpr uint32_t ID_VK = umma::idesc_bf16(DVS, DK, umma::MN_MAJOR, umma::MN_MAJOR);
#pragma unroll 1
            for (int c = 0; c < NK; ++c) {
                load_k(c);
                if (state) load_v(c);
            }
            for (int c = 0; c < n; ++c) {
                if (c > 0) {
                    if (state) {
                        wait(v_free + (c - 1) % NV, (c - 1) / NV);
                        load_v(c - 1 + NV);
                    }
                    wait(k_free + (c - 1) % NK, (c - 1) / NK);
                    load_k(c - 1 + NK);
                }
                wait(full_k + c % NK, c / NK);
                wait(vw_ready, c);
                if (c > 0) wait(ds_free, c - 1);  // the last one has been read
                umma::fence_after_sync();
                if (elect_one()) {
                    const uint64_t k0 = desc_mn + ((M::K + (c % NK) * M::QB) >> 4), w0 = desc_mn + (M::W >> 4);
#pragma unroll 1
                    for (int a = VP - 1; a >= 0; --a)  // the smallest products first
#pragma unroll
                        for (int k = 0; k < CT / 16; ++k)
                            umma::mma_bf16(tmem + M::T_DS, w0 + ((a * M::VB + 2048 * k) >> 4), k0 + (2048 * k >> 4), ID_VK, a < VP - 1 || k > 0);
                    umma::mma_commit(ds_done);
                    umma::mma_commit(k_free + c % NK);
                }
                __syncwarp();
            }
        } else if (!state) {  // O1 = P' V
            constexpr uint32_t ID_PV = umma::idesc_bf16(128, DVS, umma::K_MAJOR, umma::MN_MAJOR);
#pragma unroll 1
            for (int c = 0; c < NV; ++c) load_v(c);
            for (int c = 0; c < n; ++c) {
                if (c > 0) {
                    wait(v_free + (c - 1) % NV, (c - 1) / NV);
                    load_v(c - 1 + NV);
                }
                wait(full_v + c % NV, c / NV);
                wait(p_ready + (c & 1), c >> 1);
                if (c >= M::NO) wait(o_free + ((c - M::NO) & 1), (c - M::NO) >> 1);  // the outputs in O1's place have been read
                umma::fence_after_sync();
                if (elect_one()) {
                    const uint32_t tp = tmem + M::T_P + 128 * (c % NP);
                    const uint64_t v0 = desc_mn + ((M::V + (c % NV) * M::VB) >> 4);
#pragma unroll 1
                    for (int a = 1; a >= 0; --a)
#pragma unroll
                        for (int k = 0; k < CT / 16; ++k)
                            mma_ts(tmem + T_O1 + DVS * (c % M::NO), tp + 16 * k + 8 * a, v0 + (2048 * k >> 4), ID_PV, a < 1 || k > 0);
                    umma::mma_commit(o_done + (c & 1));
                    umma::mma_commit(v_free + c % NV);
                }
                __syncwarp();
            }
        }
        // every MMA and load issued ends before the block does
        if (elect_one()) {
            umma::mma_commit(drain + (warp - 17));
            for (uint32_t i = 0; i < kPolls && !mbar_try_wait(drain + (warp - 17), 0); ++i) {
            }
            auto landed = [&](uint64_t* full, int ring) {
                for (int c = n > ring ? n - ring : 0; c < n; ++c)
                    for (uint32_t i = 0; i < kPolls && !mbar_try_wait(full + c % ring, (c / ring) & 1); ++i) {
                    }
            };
            if (warp == 17 && !state) landed(full_q, NQ);
            if (warp == 18) landed(full_k, NK);
            if (warp == (state ? 18 : 19)) landed(full_v, NV);
        }
        __syncwarp();
    }
    umma::fence_before_sync();
    __syncthreads();
    if (warp == 16) {
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

template <int DK, int VP>
int launch(const UmmaParams& up, int64_t blocks, cudaStream_t s) {
    static std::atomic<uint64_t> done{0};
    auto kern = umma_attention_kernel<DK, VP>;
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
// map can say of the strides.  Not the scales over 2^32: the test for them in the outputs' loop alone
// took 1x16384 32x128 from 252 to 263 us.
bool umma_takes(const AttnParams& p, int64_t nb) {
    auto in = [](int64_t n, int64_t stride) { return n <= 1 || (stride > 0 && stride < (int64_t(1) << 38)); };
    for (const Stream* x : {&p.q, &p.k, &p.v})
        if (!in(p.H / x->share, x->sh) || !in(p.T, x->st) || !in(nb, x->sb)) return false;
    if (p.late != 1.0f) return false;
    return p.T < (int64_t(1) << 31) - 256 && nb < (int64_t(1) << 31) && p.ob % 8 == 0 && p.ot % 8 == 0 && p.oh % 8 == 0;
}

int umma_run(const AttnParams& p, int64_t nb, uint32_t* redo, cudaStream_t stream) {
    if (int rc = ensure_context()) return rc;
    UmmaParams up{};
    up.a = p, up.redo = redo, up.polls = umma_polls.load(std::memory_order_relaxed);
    up.wide = reinterpret_cast<uintptr_t>(p.out) % 32 == 0 && p.ob % 16 == 0 && p.ot % 16 == 0 && p.oh % 16 == 0;
    if (int rc = encode(&up.q, p.q, nb, p.T, p.H / p.q.share, p.dk)) return rc;
    if (int rc = encode(&up.k, p.k, nb, p.T, p.H / p.k.share, p.dk)) return rc;
    if (int rc = encode(&up.v, p.v, nb, p.T, p.H / p.v.share, p.dv)) return rc;
    const int64_t blocks = nb * p.H * p.slices * p.launched();
    auto go = [&](auto dk) {
        constexpr int DK = decltype(dk)::value;
        return p.sT != nullptr ? launch<DK, 3>(up, blocks, stream) : launch<DK, 2>(up, blocks, stream);
    };
    return p.dk <= 64 ? go(std::integral_constant<int, 64>{}) : go(std::integral_constant<int, 128>{});
}

}  // namespace attention
}  // namespace need

extern "C" void need_test_linear_attention_polls(uint32_t polls) { umma_polls.store(polls == 0 ? kPolls : polls, std::memory_order_relaxed); }
