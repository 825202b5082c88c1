// linear_attention.cu -- linear attention with a decay for each head
// (need_linear_attention): over whole prompts, in chunks on the tensor cores.
//
//   S_t = a_t S_{t-1} + k_t^T v_t,   o_t = scale q_t S_t,   a = exp(log_decay)
//
// With G the running sum of the log decays inside a chunk of 64 tokens and S the
// state that enters it,
//
//   o_t = scale (e^{G_t} q_t S + sum_{s <= t} e^{G_t - G_s} (q_t . k_s) v_s)
//   S'  = e^{G_end} S + sum_s e^{G_end - G_s} k_s^T v_s
//
// A marked token (or a log decay of -infinity) starts a segment: the terms that
// would cross it are left out by selection, whatever they hold.
//
// One CTA walks the chunks of one (sequence, head, 64 columns of v).  Its warps own 16
// columns each, of the outputs and of the state, which stays in their registers in
// fp32 as the accumulators of (v e^{G_end - G_s})^T k: transposed, so that the same
// registers are the B operand of q S.  The scores are computed a row block per warp
// and shared through shared memory.
//
// Precision.  The tensor cores take bf16.  An operand that is not exactly bf16 is
// given as a sum of bf16 values (planes), each the rounding of what the ones before it
// leave: 16-bit results need 2 planes of the scores and of the state (2^-17 of a
// value; one plane would add an error as large as the result's own rounding), fp32
// ones and the state itself 3 (2^-25).  f16 inputs are 2 planes exactly, fp32 ones 3;
// products of planes below the last place are left out.  Sums are fp32.  The decays'
// running sums are fp64, kept as two floats: a difference of two of them is exact to
// fp32 however far the chunk has decayed.
//
// A chunk whose q, k, v or entering state holds an infinity or NaN (or fp32 values that a
// bf16 rounding would carry over the largest), whose scores pass fp32, or whose log decays
// hold a NaN or a value over 1, is run token by token in fp32 instead: under a score of 0
// it would reach the tokens before it, and other segments, and planes of an infinity make
// a NaN of it.
//
// bf16 rows of whole 16 bytes and more than 64 tokens are linear_attention_umma.cu's (104
// chains of 64 features: 128 tokens 9.6 us there and 12.0 here, 64 tokens 9.0 and 7.6).
// Here the tensor pipe is busy a third of the time: the loads, the split into planes, the
// scores and the products with them follow one another in a chunk, some 5 us.  3 x 777
// tokens, 6 heads of 40 x 72 in fp16, in 7 segments: 32 us; 16 x 2048 tokens, 16 heads of
// 64 x 64: fp16 260 us, fp32 362 (0.5 and 0.8 TB/s).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <cmath>
#include <type_traits>

#include "host_common.h"
#include "linear_attention.cuh"
#include "need_scan.h"
#include "ptx.cuh"

using namespace need;
using namespace need::attention;

namespace {

constexpr int C = 64;       // tokens of a chunk
constexpr int kWarps = 4;   // of 16 columns of v each
constexpr int DV = 16 * kWarps;
constexpr int kThreads = 32 * kWarps;

// ------------------------------------------------------------------ pieces
__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool live) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(live ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
__device__ __forceinline__ void cp_wait_all() { asm volatile("cp.async.wait_group 0;" ::: "memory"); }

// Byte offset of 16-byte piece `piece` of row `row` in a plane of bf16 rows, 64 columns
// (128 bytes) at a time: pieces change places within 8 rows, so that ldmatrix meets every
// bank once.
__device__ __forceinline__ uint32_t at(int row, int piece) {
    return static_cast<uint32_t>((piece >> 3) * C * 128 + row * 128 + (((piece & 7) ^ (row & 7)) << 4));
}

// Planes of a type's inputs, of computed operands, and the sum of plane numbers below
// which a product counts (of the scores; of the products with the scores and the state).
template <typename T>
struct Split {
    static constexpr int IN = 1, SCORE = 2, QK = 1, OUT = 2;
};
template <>
struct Split<__half> {
    static constexpr int IN = 2, SCORE = 2, QK = 2, OUT = 2;
};
template <>
struct Split<float> {
    static constexpr int IN = 3, SCORE = 3, QK = 3, OUT = 3;
};
constexpr int kStatePlanes = 3;  // of v e^{...}: what the state sums

// f(a, b) for the planes a < NA and b < NB whose numbers sum to less than LIM, the smallest
// products first.
template <int LIM, int NA, int NB, typename F>
__device__ __forceinline__ void products(F&& f) {
#pragma unroll
    for (int sum = LIM - 1; sum >= 0; --sum)
#pragma unroll
        for (int a = 0; a < NA; ++a)
            if (a <= sum && sum - a < NB) f(a, sum - a);
}
__device__ __forceinline__ void add4(float (&x)[4], const float (&y)[4]) {
    const float2 a = __fadd2_rn(make_float2(x[0], x[1]), make_float2(y[0], y[1]));
    const float2 b = __fadd2_rn(make_float2(x[2], x[3]), make_float2(y[2], y[3]));
    x[0] = a.x, x[1] = a.y, x[2] = b.x, x[3] = b.y;
}

// A chunk's decays.
struct alignas(16) Decays {
    float hi[C], lo[C];  // log2 of the product from the chunk's first token on, as a sum
    float w[C];          // from a token to the chunk's end; 0 where a segment starts in between
    float eg[C];         // scale times that from the entering state to a token; 0 likewise
    float end[C];        // from a token to the end of its block of 16
    int seg[C];          // segments started up to the token
    float d;             // over the chunk; -1 where a segment starts in it
    int pairwise;        // scores take each pair's own decay
};

template <typename T, int DK, bool VEC>
struct Layout {
    using S = Split<T>;
    static constexpr int STAGES = S::IN == 1 && VEC ? 2 : 1;
    static constexpr int Q = 0, K = S::IN * C * DK * 2, V = 2 * K, STAGE = V + S::IN * C * DV * 2;
    static constexpr int P = STAGES * STAGE, G = P + S::SCORE * C * C * 2, BYTES = G + 2 * static_cast<int>(sizeof(Decays));
};

// ------------------------------------------------------------------ loads
// Rows [t0, t0 + C) of one tensor into its planes, 8 values of a thread at a time.  All of
// a thread's loads are issued before the first is split: one after another they cost a
// fp16 chunk 4 us.
template <typename T, int COLS, bool VEC>
struct Loader {
    static constexpr int IN = Split<T>::IN, PIECES = COLS / 8, N = C * PIECES / kThreads;
    static constexpr int W = VEC ? 8 * static_cast<int>(sizeof(T)) / 16 : 8;
    using Raw = typename std::conditional<VEC, uint4, T>::type;
    Raw raw[N][W];

    __device__ __forceinline__ void load(const T* base, int64_t st, int64_t t0, int64_t T_, int col0, int cols) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int n = i * kThreads + threadIdx.x, row = n / PIECES, col = col0 + (n % PIECES) * 8;
            const T* from = base + (t0 + row) * st + col;
#pragma unroll
            for (int w = 0; w < W; ++w) {
                const bool live = t0 + row < T_ && col + w * (8 / W) < cols;
                if constexpr (VEC) raw[i][w] = live ? __ldg(reinterpret_cast<const uint4*>(from) + w) : make_uint4(0, 0, 0, 0);
                else raw[i][w] = live ? from[w] : T(0.0f);
            }
        }
    }
    // true where a value is not finite (or too near the largest to be rounded)
    __device__ __forceinline__ bool store(char* dst) const {
        float2 chk = splat(0.0f);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int n = i * kThreads + threadIdx.x, row = n / PIECES, piece = n % PIECES;
            const T* x = reinterpret_cast<const T*>(&raw[i][0]);
            uint32_t pl[4][IN];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                split<IN>(make_float2(to_float(x[2 * e]), to_float(x[2 * e + 1])), pl[e]);
                // of a value that rounds to an infinity the first plane is one
                chk = __ffma2_rn(unpack_bf16(pl[e][0]), splat(0.0f), chk);
            }
#pragma unroll
            for (int p = 0; p < IN; ++p)
                *reinterpret_cast<uint4*>(dst + p * C * COLS * 2 + at(row, piece)) =
                    make_uint4(pl[0][p], pl[1][p], pl[2][p], pl[3][p]);
        }
        return !(chk.x == 0.0f && chk.y == 0.0f);
    }
};

// The same of bf16 rows by asynchronous copies of 16 bytes.  A thread copies one piece of
// every 16th row (of 64 columns), or of every 8th (of 128).
template <int COLS>
struct Copier {
    static constexpr int PIECES = COLS / 8, STEP = kThreads / PIECES, N = C / STEP;  // rows apart, copies
    const __nv_bfloat16* from;
    int64_t st;
    uint32_t to;  // within the plane
    int row;
    bool in;
    __device__ __forceinline__ Copier(const __nv_bfloat16* base, int64_t st_, int64_t t0, int col0, int cols) : st(st_) {
        row = threadIdx.x / PIECES;
        const int piece = threadIdx.x % PIECES, col = col0 + piece * 8;
        in = col < cols;
        to = at(row, piece);
        from = base + (in ? (t0 + row) * st + col : 0);
    }
    // rows of a chunk of `rows` of them, into the plane at dst; then on to the next chunk
    __device__ __forceinline__ void copy(uint32_t dst, const __nv_bfloat16* base, int64_t rows) {
        if (rows >= C) {
#pragma unroll
            for (int i = 0; i < N; ++i) cp_async16(dst + to + i * STEP * 128, from + i * STEP * st, in);
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const bool live = in && row + i * STEP < rows;
                cp_async16(dst + to + i * STEP * 128, live ? from + i * STEP * st : base, live);
            }
        }
        if (in) from += C * st;
    }
};
// Whether a piece that this thread has copied holds an infinity or NaN.
template <int COLS>
__device__ __forceinline__ bool check_rows(const char* src) {
    constexpr int PIECES = COLS / 8;
    const __nv_bfloat162 zero = __floats2bfloat162_rn(0.0f, 0.0f);
    __nv_bfloat162 chk = zero;
#pragma unroll
    for (int n0 = 0; n0 < C * PIECES; n0 += kThreads) {
        const int n = n0 + threadIdx.x;
        const uint4 u = *reinterpret_cast<const uint4*>(src + at(n / PIECES, n % PIECES));
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) chk = __hfma2(*reinterpret_cast<const __nv_bfloat162*>(&w[e]), zero, chk);
    }
    const float2 f = __bfloat1622float2(chk);
    return !(f.x == 0.0f && f.y == 0.0f);
}

// ------------------------------------------------------------------ decays
// A lane's two tokens of a chunk.
struct TokenPair {
    float ld[2];
    bool reset[2];
};
__device__ __forceinline__ TokenPair load_decays(const AttnParams& p, const float* ld, const uint8_t* seg, int64_t t0) {
    TokenPair r;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        const int64_t t = t0 + 2 * (threadIdx.x & 31) + e;
        const bool live = t < p.T;
        const float x = live ? ld[t * p.lt] : 0.0f;
        r.reset[e] = (live && seg != nullptr && seg[t * p.gt] != 0) || x == -INFINITY;
        // a token's state falls below every fp32 value long before e^-10000; a NaN stays one
        r.ld[e] = r.reset[e] ? 0.0f : x < -10000.0f ? -10000.0f : x;
    }
    return r;
}
// One warp: the chunk's running sums from its 64 log decays.  True where one of them is no
// number or so far above 0 that a product of 64 leaves fp32's range.
__device__ __forceinline__ bool make_decays(const TokenPair& tp, float scale, Decays& g) {
    const int lane = threadIdx.x & 31;
    const double x0 = static_cast<double>(tp.ld[0]) * 1.4426950408889634074, x1 = static_cast<double>(tp.ld[1]) * 1.4426950408889634074;
    double incl = x0 + x1;
#pragma unroll
    for (int m = 1; m < 32; m <<= 1) {
        const double o = __shfl_up_sync(0xffffffffu, incl, m);
        if (lane >= m) incl += o;
    }
    double before = __shfl_up_sync(0xffffffffu, incl, 1);
    if (lane == 0) before = 0.0;
    const uint32_t m0 = __ballot_sync(0xffffffffu, tp.reset[0]), m1 = __ballot_sync(0xffffffffu, tp.reset[1]);
    const uint32_t lt = (1u << lane) - 1u;
    const double G[2] = {before + x0, incl};
    int s[2];
    s[0] = __popc(m0 & lt) + __popc(m1 & lt) + (tp.reset[0] ? 1 : 0);
    s[1] = s[0] + (tp.reset[1] ? 1 : 0);
    const double end = __shfl_sync(0xffffffffu, incl, 31), block_end = __shfl_sync(0xffffffffu, incl, lane | 7);
    const int send = __popc(m0) + __popc(m1);
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        const int i = 2 * lane + e;
        const float hi = static_cast<float>(G[e]);
        g.hi[i] = hi, g.lo[i] = static_cast<float>(G[e] - hi);
        g.seg[i] = s[e];
        g.w[i] = s[e] == send ? ex2(static_cast<float>(end - G[e])) : 0.0f;
        g.eg[i] = s[e] == 0 ? scale * ex2(hi) : 0.0f;
        g.end[i] = ex2(static_cast<float>(block_end - G[e]));
    }
    // A block's column factor may fall to 0 where a pair's decay does not, if states grow after it: then
    // (2^60 and more between two tokens' sums, one of them growing), and where a segment starts.
    const bool grows = __any_sync(0xffffffffu, tp.ld[0] > 0.0f || tp.ld[1] > 0.0f);
    const bool wide = __any_sync(0xffffffffu, fabs(G[0] - end) > 30.0 || fabs(G[1] - end) > 30.0);
    if (lane == 0) g.d = send == 0 ? ex2(static_cast<float>(end)) : -1.0f, g.pairwise = send != 0 || (grows && wide) ? 1 : 0;
    return __any_sync(0xffffffffu, !(tp.ld[0] <= 1.0f && tp.ld[1] <= 1.0f));
}
// ------------------------------------------------------------------ the kernel
// What a launch's segments are run for.
enum Kind { OUTPUTS, STATES, MIXED };

// A chunk token by token, in fp32, from the inputs themselves; s as in attention_kernel, jw the warp's
// first column.  Its registers are its own: inlined it took 16x2048 16x64 f32 from 362 to 397 us.
template <typename T, int NI>
__device__ __noinline__ void run_by_token(const AttnParams& p, float (&s)[NI][4], const T* q, const T* k, const T* v, const float* ld,
                                          const uint8_t* marks, T* out, int64_t t0, int jw, bool state) {
    const int lane = threadIdx.x & 31, g = lane >> 2, c2 = (lane & 3) * 2;
    const int n = static_cast<int>(p.T - t0 < C ? p.T - t0 : C);
    for (int r = 0; r < n; ++r) {
        const int64_t t = t0 + r;
        const bool reset = starts(ld, p.lt, marks, p.gt, t);
        const float a = expf(ld[t * p.lt]);
        const int j = jw + g;
        const float v0 = j < p.dv ? to_float(v[t * p.v.st + j]) : 0.0f;
        const float v1 = j + 8 < p.dv ? to_float(v[t * p.v.st + j + 8]) : 0.0f;
        float o0 = 0.0f, o1 = 0.0f;
#pragma unroll
        for (int m = 0; m < NI; ++m)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int i = 8 * m + c2 + e;
                if (i < p.dk) {
                    const float kk = to_float(k[t * p.k.st + i]);
                    s[m][e] = reset ? kk * v0 : fmaf(a, s[m][e], kk * v0);
                    s[m][2 + e] = reset ? kk * v1 : fmaf(a, s[m][2 + e], kk * v1);
                    if (!state) {
                        const float qq = to_float(q[t * p.q.st + i]);
                        o0 = fmaf(qq, s[m][e], o0), o1 = fmaf(qq, s[m][2 + e], o1);
                    }
                }
            }
        if (!state) {
#pragma unroll
            for (int m = 1; m < 4; m <<= 1) {
                o0 += __shfl_xor_sync(0xffffffffu, o0, m);
                o1 += __shfl_xor_sync(0xffffffffu, o1, m);
            }
            if (c2 == 0 && j < p.dv) out[t * p.ot + j] = static_cast<T>(p.scale * p.late * o0);
            if (c2 == 2 && j + 8 < p.dv) out[t * p.ot + j + 8] = static_cast<T>(p.scale * p.late * o1);
        }
    }
}

template <typename T, int DK, bool VEC, int KIND>
__global__ void __launch_bounds__(kThreads, DK == 64 && Split<T>::IN < 3 ? 3 : 2) attention_kernel(const __grid_constant__ AttnParams p) {
    using S = Split<T>;
    using L = Layout<T, DK, VEC>;
    constexpr int NI = DK / 8;  // 8-feature tiles of the state
    constexpr int MQ = S::IN == 1 ? 4 : 2;  // row blocks whose products with the state run side by side
    constexpr bool FRESH = S::IN == 3;      // fp32: partial sums apart, as for the state
    extern __shared__ __align__(128) char smem[];
    if (p.redo != nullptr && p.redo[blockIdx.x] == 0) return;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c2 = (lane & 3) * 2;
    int64_t id = blockIdx.x;
    const int segs = p.launched(), seg = static_cast<int>(id % segs) + (p.ahead ? 0 : p.lead);
    const bool state = KIND == MIXED ? seg >= p.lead : KIND == STATES;  // only the state
    id /= segs;
    const int slice = static_cast<int>(id % p.slices);
    const int64_t chain = id / p.slices;
    const int64_t b = chain / p.H;
    const int h = static_cast<int>(chain % p.H), col0 = slice * DV, jw = col0 + 16 * warp;
    const T* q = static_cast<const T*>(p.q.p) + b * p.q.sb + (h / p.q.share) * p.q.sh;
    const T* k = static_cast<const T*>(p.k.p) + b * p.k.sb + (h / p.k.share) * p.k.sh;
    const T* v = static_cast<const T*>(p.v.p) + b * p.v.sb + (h / p.v.share) * p.v.sh;
    const float* ld = p.ld + b * p.lb + h * p.lh;
    const uint8_t* marks = p.seg == nullptr ? nullptr : p.seg + b * p.gb;
    T* out = static_cast<T*>(p.out) + b * p.ob + h * p.oh;
    const int64_t chunks = (p.T + C - 1) / C, c0 = p.segment(seg), c1 = p.segment(seg + 1) < chunks ? p.segment(seg + 1) : chunks;
    Decays* const gates = reinterpret_cast<Decays*>(smem + L::G);
    const uint32_t sm = smem_addr(smem);

    // the state, transposed: rows j = jw + g and + 8, columns i = 8 n + c2 and + 1
    float s[NI][4];
    bool entered;
    {
        const float* from = state ? nullptr : seg > 0 ? p.part + (chain * (p.nseg - 1) + seg - 1) * p.dk * int64_t(p.dv)
                                  : p.s0 != nullptr   ? p.s0 + chain * p.dk * int64_t(p.dv) : nullptr;
        const bool fresh = from != nullptr && starts(ld, p.lt, marks, p.gt, c0 * C);  // nothing of it is seen
        entered = from != nullptr;
#pragma unroll
        for (int n = 0; n < NI; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int i = 8 * n + c2 + (e & 1), j = jw + g + (e >> 1) * 8;
                s[n][e] = from != nullptr && i < p.dk && j < p.dv ? from[int64_t(i) * p.dv + j] : 0.0f;
            }
        if (fresh)
#pragma unroll
            for (int n = 0; n < NI; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.0f;
    }
    // Whether the state holds an infinity or NaN (2^-8 more of a value rounds to one): after finite
    // chunks it does not.
    auto not_finite = [&] {
        float chk = 0.0f;
#pragma unroll
        for (int n = 0; n < NI; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) chk = fmaf((1.0f + 0x1p-8f) * s[n][e], 0.0f, chk);
        return !(chk == 0.0f);
    };
    bool lost = entered && not_finite();
    double total = 1.0;  // the segment's decay

    using B16 = __nv_bfloat16;
    const B16 *qc = reinterpret_cast<const B16*>(q), *kc = reinterpret_cast<const B16*>(k), *vc = reinterpret_cast<const B16*>(v);
    Copier<DK> copy_q(qc, p.q.st, c0 * C, 0, p.dk), copy_k(kc, p.k.st, c0 * C, 0, p.dk);
    Copier<DV> copy_v(vc, p.v.st, c0 * C, col0, p.dv);
    auto issue = [&](int64_t c) {  // the asynchronous copies of a chunk, in turn
        if constexpr (L::STAGES == 2) {
            const uint32_t to = sm + (c & 1) * L::STAGE;
            if (!state) copy_q.copy(to + L::Q, qc, p.T - c * C);
            copy_k.copy(to + L::K, kc, p.T - c * C);
            copy_v.copy(to + L::V, vc, p.T - c * C);
            cp_commit();
        }
    };
    issue(c0);
    bool wild = false;  // warp 0: of the next chunk's decays
    bool again = false;  // the chunk is run a second time, token by token
    TokenPair next{};
    if (warp == 0) wild = make_decays(load_decays(p, ld, marks, c0 * C), p.scale, gates[c0 & 1]);

    for (int64_t c = c0; c < c1; ++c) {
        const int64_t t0 = c * C;
        const int stage = L::STAGES == 2 ? static_cast<int>(c & 1) : 0;
        char* const buf = smem + stage * L::STAGE;
        const uint32_t sbuf = sm + stage * L::STAGE;
        bool bad;
        if constexpr (L::STAGES == 2) {
            cp_wait_all();
            bad = check_rows<DK>(buf + L::K) | check_rows<DV>(buf + L::V);
        } else {
            constexpr bool ALL = DK == 64 || S::IN < 3;  // else the registers hold K and V only
            Loader<T, DK, VEC> lk, lq;
            Loader<T, DV, VEC> lv;
            lk.load(k, p.k.st, t0, p.T, 0, p.dk), lv.load(v, p.v.st, t0, p.T, col0, p.dv);
            if (!state && ALL) lq.load(q, p.q.st, t0, p.T, 0, p.dk);
            __syncthreads();  // the chunk before this one has been read
            bad = lk.store(buf + L::K) | lv.store(buf + L::V);
            if (!state && !ALL) lq.load(q, p.q.st, t0, p.T, 0, p.dk);
            if (!state) lq.store(buf + L::Q);
        }
        bad |= lost;
        bad = __syncthreads_or(bad | wild);  // the chunk and its decays are there
        const Decays& gt = gates[c & 1];
        if (c + 1 < c1 && !again) {
            issue(c + 1);
            if (warp == 0) next = load_decays(p, ld, marks, t0 + C);
        }
        auto by_token = [&] {
            float x[NI][4];
#pragma unroll
            for (int n = 0; n < NI; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) x[n][e] = s[n][e];
            run_by_token<T, NI>(p, x, q, k, v, ld, marks, out, t0, jw, state);
#pragma unroll
            for (int n = 0; n < NI; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) s[n][e] = x[n][e];
            lost = not_finite();
        };
        if (KIND != OUTPUTS && !again) total = total == -1.0 || gt.d == -1.0f ? -1.0 : total * gt.d;

        if (bad || again) {
            by_token();
            if (warp == 0 && c + 1 < c1 && !again) wild = make_decays(next, p.scale, gates[(c + 1) & 1]);
            again = false;
            continue;
        }

        // rows and pieces of this lane's ldmatrix addresses: 16 rows x 16 columns a load
        const int lr = lane & 15, lp = lane >> 4;                              // [m][k] tiles, and [k][n] ones transposed
        const int br = (lane & 7) + ((lane >> 4) << 3), bp = (lane >> 3) & 1;  // [n][k] tiles, and [k][m] ones transposed
        const bool resets = gt.d == -1.0f;
        float o[4][2][4] = {};
        float2 over = splat(0.0f);  // 0 unless a score is no finite number (one past fp32, or q holds none)
        if (!state) {
            // the scores on and below the diagonal, in blocks of 16 x 16: each warp the one on
            // the diagonal and one or two others
            for (int i = 0; i < (warp == 1 || warp == 2 ? 3 : 2); ++i) {
                const int rb = i == 0 || warp == 2 || (warp == 1 && i == 1) ? warp : 3;
                const int cb = i == 0 ? warp : warp == 3 ? 2 : warp == 0 ? 0 : i == 1 ? 0 : 1;
                float acc[2][2][4] = {};  // [steps taken in turn][8 tokens]
#pragma unroll
                for (int ks = 0; ks < DK / 16; ++ks) {
                    uint32_t qa[S::IN][4], kb[S::IN][4];
#pragma unroll
                    for (int a = 0; a < S::IN; ++a) {
                        ldsm4(qa[a], sbuf + L::Q + a * C * DK * 2 + at(16 * rb + lr, 2 * ks + lp));
                        ldsm4(kb[a], sbuf + L::K + a * C * DK * 2 + at(16 * cb + br, 2 * ks + bp));
                    }
                    products<S::QK, S::IN, S::IN>([&](int a, int b2) {
                        mma(acc[ks & 1][0], qa[a], kb[b2][0], kb[b2][1]);
                        mma(acc[ks & 1][1], qa[a], kb[b2][2], kb[b2][3]);
                    });
                }
                const int r0 = 16 * rb + g;
                const float h0 = gt.hi[r0], l0 = gt.lo[r0], h1 = gt.hi[r0 + 8], l1 = gt.lo[r0 + 8];
                const bool pairwise = rb == cb || gt.pairwise != 0;
                float f0 = 0.0f, f1 = 0.0f;  // of a block below the diagonal: from its columns' end on
                if (!pairwise) {
                    const float he = gt.hi[16 * cb + 15], le = gt.lo[16 * cb + 15];
                    f0 = p.scale * ex2((h0 - he) + (l0 - le)), f1 = p.scale * ex2((h1 - he) + (l1 - le));
                }
#pragma unroll
                for (int n = 0; n < 2; ++n) {
                    const int col = 16 * cb + 8 * n + c2;
                    float2 x0 = make_float2(acc[0][n][0] + acc[1][n][0], acc[0][n][1] + acc[1][n][1]);
                    float2 x1 = make_float2(acc[0][n][2] + acc[1][n][2], acc[0][n][3] + acc[1][n][3]);
                    if (!pairwise) {
                        const float2 end = *reinterpret_cast<const float2*>(&gt.end[col]);
                        x0 = __fmul2_rn(x0, __fmul2_rn(end, splat(f0)));
                        x1 = __fmul2_rn(x1, __fmul2_rn(end, splat(f1)));
                    } else {
                        const int s0 = gt.seg[r0], s1 = gt.seg[r0 + 8];
                        const float2 hs = *reinterpret_cast<const float2*>(&gt.hi[col]), ls = *reinterpret_cast<const float2*>(&gt.lo[col]);
                        const int2 ss = *reinterpret_cast<const int2*>(&gt.seg[col]);
                        x0.x = ss.x == s0 && col <= r0 ? x0.x * (p.scale * ex2((h0 - hs.x) + (l0 - ls.x))) : 0.0f;
                        x0.y = ss.y == s0 && col + 1 <= r0 ? x0.y * (p.scale * ex2((h0 - hs.y) + (l0 - ls.y))) : 0.0f;
                        x1.x = ss.x == s1 && col <= r0 + 8 ? x1.x * (p.scale * ex2((h1 - hs.x) + (l1 - ls.x))) : 0.0f;
                        x1.y = ss.y == s1 && col + 1 <= r0 + 8 ? x1.y * (p.scale * ex2((h1 - hs.y) + (l1 - ls.y))) : 0.0f;
                    }
                    over = __ffma2_rn(x0, splat(0.0f), over), over = __ffma2_rn(x1, splat(0.0f), over);
                    uint32_t p0[S::SCORE], p1[S::SCORE];
                    split<S::SCORE>(x0, p0);
                    split<S::SCORE>(x1, p1);
#pragma unroll
                    for (int a = 0; a < S::SCORE; ++a) {
                        char* const to = smem + L::P + a * C * C * 2 + c2 * 2;
                        *reinterpret_cast<uint32_t*>(to + at(r0, 2 * cb + n)) = p0[a];
                        *reinterpret_cast<uint32_t*>(to + at(r0 + 8, 2 * cb + n)) = p1[a];
                    }
                }
            }
            // what the entering state gives: all 64 rows, this warp's 16 columns
#pragma unroll
            for (int ks = 0; ks < DK / 16; ++ks) {
                uint32_t sb0[2][S::SCORE], sb1[2][S::SCORE];  // [column tile][plane], features 0-7 and 8-15 of the step
#pragma unroll
                for (int n = 0; n < 2; ++n) {
                    split<S::SCORE>(make_float2(s[2 * ks][2 * n], s[2 * ks][2 * n + 1]), sb0[n]);
                    split<S::SCORE>(make_float2(s[2 * ks + 1][2 * n], s[2 * ks + 1][2 * n + 1]), sb1[n]);
                }
#pragma unroll
                for (int m0 = 0; m0 < 4; m0 += MQ) {
                    uint32_t qf[MQ][S::IN][4];
#pragma unroll
                    for (int m = 0; m < MQ; ++m)
#pragma unroll
                        for (int a = 0; a < S::IN; ++a)
                            ldsm4(qf[m][a], sbuf + L::Q + a * C * DK * 2 + at(16 * (m0 + m) + lr, 2 * ks + lp));
                    float t[MQ][2][4] = {};
                    products<S::OUT, S::IN, S::SCORE>([&](int a, int b2) {
#pragma unroll
                        for (int m = 0; m < MQ; ++m)
#pragma unroll
                            for (int n = 0; n < 2; ++n) mma(FRESH ? t[m][n] : o[m0 + m][n], qf[m][a], sb0[n][b2], sb1[n][b2]);
                    });
                    if (FRESH)
#pragma unroll
                        for (int m = 0; m < MQ; ++m)
#pragma unroll
                            for (int n = 0; n < 2; ++n) add4(o[m0 + m][n], t[m][n]);
                }
            }
#pragma unroll
            for (int m = 0; m < 4; ++m)
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    const int row = 16 * m + g + 8 * r;
                    const float eg = gt.eg[row];
                    const bool reach = !resets || gt.seg[row] == 0;
#pragma unroll
                    for (int n = 0; n < 2; ++n)
#pragma unroll
                        for (int e = 0; e < 2; ++e) o[m][n][2 * r + e] = reach ? eg * o[m][n][2 * r + e] : 0.0f;
                }
        }
        if (warp == 0 && c + 1 < c1) wild = make_decays(next, p.scale, gates[(c + 1) & 1]);
        if (!state && __syncthreads_or(!(over.x == 0.0f && over.y == 0.0f))) {  // the scores are there
            again = true, --c;
            continue;
        }

        // the scores times v, and the state
        if (resets) {
#pragma unroll
            for (int n = 0; n < NI; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.0f;
        } else {
            const float2 d = splat(gt.d);
#pragma unroll
            for (int n = 0; n < NI; ++n) {
                const float2 x = __fmul2_rn(make_float2(s[n][0], s[n][1]), d), y = __fmul2_rn(make_float2(s[n][2], s[n][3]), d);
                s[n][0] = x.x, s[n][1] = x.y, s[n][2] = y.x, s[n][3] = y.y;
            }
        }
#pragma unroll
        for (int kb = 0; kb < 4; ++kb) {  // blocks of 16 tokens
            uint32_t vf[S::IN][4];  // (tokens 0-7, columns 0-7), (0-7, 8-15), (8-15, 0-7), (8-15, 8-15)
#pragma unroll
            for (int a = 0; a < S::IN; ++a) ldsm4_t(vf[a], sbuf + L::V + a * C * DV * 2 + at(16 * kb + br, 2 * warp + bp));
            if (!state) {
                float t[4][2][4] = {};
                products<S::OUT, S::SCORE, S::IN>([&](int a, int b2) {
#pragma unroll
                    for (int m = kb; m < 4; ++m) {
                        uint32_t pf[4];
                        ldsm4(pf, sm + L::P + a * C * C * 2 + at(16 * m + lr, 2 * kb + lp));
                        mma(FRESH ? t[m][0] : o[m][0], pf, vf[b2][0], vf[b2][2]);
                        mma(FRESH ? t[m][1] : o[m][1], pf, vf[b2][1], vf[b2][3]);
                    }
                });
                if (FRESH)
#pragma unroll
                    for (int m = kb; m < 4; ++m) add4(o[m][0], t[m][0]), add4(o[m][1], t[m][1]);
            }
            uint32_t vw[kStatePlanes][4];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float2 w = *reinterpret_cast<const float2*>(&gt.w[16 * kb + (r >> 1) * 8 + c2]);
                float2 x = unpack_bf16(vf[S::IN - 1][r]);
#pragma unroll
                for (int a = S::IN - 2; a >= 0; --a) x = __fadd2_rn(x, unpack_bf16(vf[a][r]));  // the input itself
                uint32_t pl[kStatePlanes];
                split<kStatePlanes>(__fmul2_rn(w, x), pl);
#pragma unroll
                for (int a = 0; a < kStatePlanes; ++a) vw[a][r] = pl[a];
            }
            // 16 tokens' part of the state is summed apart and added by rounding: the tensor
            // cores' own additions cut, and a long sum of one sign would drift
#pragma unroll
            for (int n0 = 0; n0 < NI; n0 += 4) {  // 32 features each
                uint32_t kf[2][S::IN][4];
#pragma unroll
                for (int n = 0; n < 2; ++n)
#pragma unroll
                    for (int b2 = 0; b2 < S::IN; ++b2)
                        ldsm4_t(kf[n][b2], sbuf + L::K + b2 * C * DK * 2 + at(16 * kb + lr, n0 + 2 * n + lp));
                float t[4][4] = {};
                products<kStatePlanes, kStatePlanes, S::IN>([&](int a, int b2) {
#pragma unroll
                    for (int n = 0; n < 2; ++n) {
                        mma(t[2 * n], vw[a], kf[n][b2][0], kf[n][b2][1]);
                        mma(t[2 * n + 1], vw[a], kf[n][b2][2], kf[n][b2][3]);
                    }
                });
#pragma unroll
                for (int n = 0; n < 4; ++n) add4(s[n0 + n], t[n]);
            }
        }
        if (!state) {
            const int64_t rows = p.T - t0;
            T* const row0 = out + t0 * p.ot + jw + c2;
#pragma unroll
            for (int m = 0; m < 4; ++m)
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    const int row = 16 * m + g + 8 * r;
                    if (row < rows)
#pragma unroll
                        for (int n = 0; n < 2; ++n) {
                            const int j = jw + 8 * n + c2;
                            const float x = p.late * o[m][n][2 * r], y = p.late * o[m][n][2 * r + 1];
                            T* const to = row0 + row * p.ot + 8 * n;
                            if (VEC) {  // whole pairs, aligned
                                if (j < p.dv) {
                                    if constexpr (sizeof(T) == 4) *reinterpret_cast<float2*>(to) = make_float2(x, y);
                                    else if constexpr (std::is_same<T, __half>::value) *reinterpret_cast<__half2*>(to) = __floats2half2_rn(x, y);
                                    else *reinterpret_cast<uint32_t*>(to) = pack_bf16(x, y);
                                }
                            } else {
                                if (j < p.dv) to[0] = static_cast<T>(x);
                                if (j + 1 < p.dv) to[1] = static_cast<T>(y);
                            }
                        }
                }
        }
    }

    float* const to = KIND != OUTPUTS ? p.part + (chain * (p.nseg - 1) + seg) * p.dk * int64_t(p.dv)
                            : seg == p.nseg - 1 && p.sT != nullptr ? p.sT + chain * p.dk * int64_t(p.dv) : nullptr;
    if (to != nullptr) {
#pragma unroll
        for (int n = 0; n < NI; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int i = 8 * n + c2 + (e & 1), j = jw + g + (e >> 1) * 8;
                if (i < p.dk && j < p.dv) to[int64_t(i) * p.dv + j] = s[n][e];
            }
    }
    if (KIND != OUTPUTS && slice == 0 && threadIdx.x == 0) put_decay(p.part_d + 2 * (chain * (p.nseg - 1) + seg), total);
}

// The state that enters each segment after the first, in the place of the own state of
// the one before it (lead: the second's lies there).
__global__ void __launch_bounds__(256) enter_kernel(const AttnParams p) {
    const int64_t n = p.dk * int64_t(p.dv), chain = blockIdx.x;
    const int64_t i = blockIdx.y * int64_t(256) + threadIdx.x;
    if (i >= n) return;
    float* s = p.part + chain * (p.nseg - 1) * n + i;
    const float* d = p.part_d + 2 * chain * (p.nseg - 1);
    float x = p.lead ? s[0] : p.s0 != nullptr ? p.s0[chain * n + i] : 0.0f;
    constexpr int B = 8;  // loads in flight
    for (int k0 = p.lead; k0 < p.nseg - 1; k0 += B) {
        float own[B];
        float2 by[B];
#pragma unroll
        for (int e = 0; e < B; ++e) {
            const int k = k0 + e < p.nseg - 1 ? k0 + e : k0;
            own[e] = s[k * n], by[e] = make_float2(d[2 * k], d[2 * k + 1]);
        }
#pragma unroll
        for (int e = 0; e < B; ++e)
            if (k0 + e < p.nseg - 1) {
                x = times_state(by[e], x) + own[e];
                s[(k0 + e) * n] = x;
            }
    }
}

// ------------------------------------------------------------------ host
struct Plan {
    bool umma;  // sm_100a's tensor cores take it, in chunks of 128
    int64_t chains, chunks;
    int32_t slices, nseg, lead;
    int64_t first_chunks, seg_chunks;  // of the first segment, of the others
};
// CTAs of attention_kernel that a multiprocessor holds (registers for 3, 227 KB).
template <typename T>
constexpr int held(bool small) {
    const int bytes = (small ? Layout<T, 64, true>::BYTES : Layout<T, 128, true>::BYTES) + 1024;
    return std::min(3, 227 * 1024 / bytes);
}
// Where there are few chains they are cut into segments, as many as the GPU holds at once (of
// umma's CTAs one a multiprocessor): all but the last are run for the state that they leave, a
// launch joins those, then all are run for the outputs.  That is worth it where it saves more
// chunks in a row than the two more launches cost (1.5 of attention_kernel's, five of umma's
// 128 tokens; a chunk for the state alone counts as 0.8).  Uncut and cut: 4 bf16 chains of 64
// features 13.8 and 17.7 us at 512 tokens, 20.7 and 17.8 at 1024; 64 fp16 ones 14.2 and 17.8
// at 128 tokens, 24.8 and 22.3 at 256, 401 and 181 at 4096; 104 fp32 ones 540 and 482 at 4096.
// umma may also run one segment more, the first for its outputs ahead (lead): of two places a
// chain, 1x16384 32x128 takes 264 us, 341 without and 350 uncut, 52 chains of 64 features at
// 4096 tokens 67, 73 without (and uncut).  (In attention_kernel the choice at run time cost more:
// 8 x 1024 tokens, 13 heads of 128 x 128 in fp32, 431 us, 391 without.)
Plan plan(bool umma, int32_t dtype, int64_t nb, int64_t T, int64_t H, int64_t dk, int64_t dv) {
    Plan pl{};
    pl.umma = umma;
    pl.chains = nb * H, pl.chunks = (T + C - 1) / C, pl.slices = int32_t((dv + DV - 1) / DV);
    const bool small = dk <= 64;
    const int64_t ctas = std::max<int64_t>(1, pl.chains * pl.slices), unit = umma ? 2 : 1, chunks = (pl.chunks + unit - 1) / unit;
    const int64_t places = 148 * (umma ? 1 : dtype == NEED_F32 ? held<float>(small) : dtype == NEED_BF16 ? held<__nv_bfloat16>(small) : held<__half>(small));
    const int64_t most = std::max<int64_t>(1, places / ctas), nseg = std::min(most, chunks), len = (chunks + nseg - 1) / nseg;
    int64_t cost = 18 * len + (umma ? 50 : 15);  // tenths of a chunk
    pl.nseg = 1, pl.first_chunks = pl.seg_chunks = chunks * unit;
    if (cost <= 10 * chunks) pl.nseg = int32_t((chunks + len - 1) / len), pl.first_chunks = pl.seg_chunks = len * unit;
    else cost = 10 * chunks;
    if (umma) {
        const int64_t n = (10 * chunks + 10 * most + 6) / (10 * most + 7), others = std::min(most, (chunks - 1) / n), first = chunks - others * n;
        if (others > 1 && std::max(10 * first, 8 * n) + 10 * n + 50 < cost)
            pl.lead = 1, pl.nseg = int32_t(others) + 1, pl.first_chunks = first * unit, pl.seg_chunks = n * unit;
    }
    return pl;
}
size_t workspace_of(const Plan& pl, int64_t dk, int64_t dv) {
    return 16 + size_t(pl.chains) * size_t(pl.nseg - 1) * (size_t(dk) * size_t(dv) + 2) * 4 + (pl.umma ? size_t(pl.chains) * pl.slices * pl.nseg * 4 : 0);
}

template <typename T, int DK, bool VEC, int KIND>
int launch(const AttnParams& p, const Plan& pl, cudaStream_t s) {
    static std::atomic<uint64_t> done{0};
    auto kern = attention_kernel<T, DK, VEC, KIND>;
    constexpr int bytes = Layout<T, DK, VEC>::BYTES;
    cudaError_t e = ensure_smem(kern, bytes, done);
    if (e != cudaSuccess) return cuda_fail(e, "linear attention shared memory");
    kern<<<static_cast<unsigned>(pl.chains * pl.slices * p.launched()), kThreads, bytes, s>>>(p);
    e = cudaGetLastError();
    return e == cudaSuccess ? NEED_OK : cuda_fail(e, "linear attention launch");
}

template <typename T, int DK, bool VEC>
int run(AttnParams p, const Plan& pl, int64_t nb, uint32_t* redo, cudaStream_t s) {
    auto part = [&](bool ahead) {
        p.ahead = ahead;
        if (pl.umma) {
            if (int rc = umma_run(p, nb, redo, s)) return rc;
        }
        // or what umma has left
        if constexpr (VEC && std::is_same<T, __nv_bfloat16>::value)
            if (ahead && p.lead) return launch<T, DK, VEC, MIXED>(p, pl, s);
        return ahead ? launch<T, DK, VEC, STATES>(p, pl, s) : launch<T, DK, VEC, OUTPUTS>(p, pl, s);
    };
    p.redo = pl.umma ? redo : nullptr;
    if (pl.nseg > 1) {
        if (int rc = part(true)) return rc;
        const dim3 grid(static_cast<unsigned>(pl.chains), static_cast<unsigned>((int64_t(p.dk) * p.dv + 255) / 256));
        enter_kernel<<<grid, 256, 0, s>>>(p);
        const cudaError_t e = cudaGetLastError();
        if (e != cudaSuccess) return cuda_fail(e, "linear attention launch");
    }
    return part(false);
}

}  // namespace

extern "C" {

size_t need_linear_attention_workspace_size(int32_t dtype, int64_t nb, int64_t T, int64_t H, int64_t dk, int64_t dv) {
    if (!dtype_ok(dtype) || nb < 1 || T < 1 || H < 1 || dk < 1 || dv < 1) return 16;
    size_t n = workspace_of(plan(false, dtype, nb, T, H, dk, dv), dk, dv);
    if (dtype == NEED_BF16) n = std::max(n, workspace_of(plan(true, dtype, nb, T, H, dk, dv), dk, dv));
    return n;
}

int need_linear_attention(const need_linear_attention_args* a, need_stream_t stream) {
    if (a == nullptr) return fail(NEED_ERR_INVALID, "linear attention: args is null");
    if (!dtype_ok(a->dtype)) return fail(NEED_ERR_UNSUPPORTED, "linear attention: dtype %d", a->dtype);
    if (a->nb < 1 || a->T < 1 || a->H < 1 || a->dk < 1 || a->dv < 1)
        return fail(NEED_ERR_INVALID, "linear attention: sizes must be positive");
    if (a->dk > NEED_LINEAR_ATTENTION_MAX_DK || a->dv > (1 << 20) || a->H > (1 << 24) || a->T > (int64_t(1) << 36))
        return fail(NEED_ERR_UNSUPPORTED, "linear attention: at most %d features a head (got %lld), sizes out of range",
                    NEED_LINEAR_ATTENTION_MAX_DK, static_cast<long long>(a->dk));
    const need_heads* in[3] = {&a->q, &a->k, &a->v};
    for (const need_heads* x : in) {
        if (x->ptr == nullptr) return fail(NEED_ERR_INVALID, "linear attention: an input is null");
        if (x->heads < 1 || a->H % x->heads != 0)
            return fail(NEED_ERR_INVALID, "linear attention: heads must divide H = %lld", static_cast<long long>(a->H));
    }
    if (a->log_decay == nullptr || a->out == nullptr) return fail(NEED_ERR_INVALID, "linear attention: log_decay and out are required");
    if (a->T > 1 && a->out_stride_t < a->dv) return fail(NEED_ERR_INVALID, "linear attention: the output's rows overlap");
    if (a->nb > (int64_t(1) << 30) / a->H / ((a->dv + DV - 1) / DV))
        return fail(NEED_ERR_UNSUPPORTED, "linear attention: too many sequences and heads");
    // parts, and blocks that are run again, read the state after final_state has been written
    const uintptr_t before = reinterpret_cast<uintptr_t>(a->state), after = reinterpret_cast<uintptr_t>(a->final_state);
    const size_t bytes = size_t(a->nb) * a->H * a->dk * a->dv * sizeof(float);
    if (before != 0 && after != 0 && before < after + bytes && after < before + bytes)
        return fail(NEED_ERR_INVALID, "linear attention: state and final_state overlap");
    const int es = dtype_bytes(a->dtype), per = 16 / es;
    AttnParams p{};
    Stream* to[3] = {&p.q, &p.k, &p.v};
    // whole 16-byte pieces: of the rows of all inputs, and pairs of the output
    bool vec = a->dk % per == 0 && a->dv % per == 0;
    for (int n = 0; n < 3; ++n) {
        const need_heads& x = *in[n];
        *to[n] = Stream{x.ptr, x.stride_b, x.stride_t, x.stride_h, int32_t(a->H / x.heads)};
        vec = vec && aligned16(x.ptr) && (x.stride_t % per == 0 || a->T == 1) && (x.stride_b % per == 0 || a->nb == 1) &&
              (x.stride_h % per == 0 || x.heads == 1);
    }
    vec = vec && aligned16(a->out) && a->out_stride_t % 2 == 0 && a->out_stride_b % 2 == 0 && a->out_stride_h % 2 == 0;
    p.ld = a->log_decay, p.lb = a->ld_stride_b, p.lt = a->ld_stride_t, p.lh = a->ld_stride_h;
    p.seg = a->seg_start, p.gb = a->seg_stride_b, p.gt = a->seg_stride_t;
    p.s0 = a->state, p.sT = a->final_state;
    p.out = a->out, p.ob = a->out_stride_b, p.ot = a->out_stride_t, p.oh = a->out_stride_h;
    p.T = a->T, p.H = int32_t(a->H), p.dk = int32_t(a->dk), p.dv = int32_t(a->dv);
    const bool large = std::fabs(a->scale) > 0x1p32f;
    p.scale = large ? 1.0f : a->scale, p.late = large ? a->scale : 1.0f;
    const Plan pl = plan(vec && a->dtype == NEED_BF16 && a->T > C && umma_takes(p, a->nb), a->dtype, a->nb, a->T, a->H,
                         a->dk, a->dv);
    if ((pl.nseg > 1 || pl.umma) && (a->workspace == nullptr || (reinterpret_cast<uintptr_t>(a->workspace) & 3u) != 0 ||
                                     a->workspace_bytes < workspace_of(pl, a->dk, a->dv)))
        return fail(NEED_ERR_WORKSPACE, "linear attention: workspace missing, misaligned or too small");
    p.slices = pl.slices, p.nseg = pl.nseg, p.lead = pl.lead, p.first_chunks = pl.first_chunks, p.seg_chunks = pl.seg_chunks;
    p.part = static_cast<float*>(a->workspace);
    p.part_d = p.part + pl.chains * (pl.nseg - 1) * a->dk * a->dv;
    uint32_t* redo = reinterpret_cast<uint32_t*>(p.part_d + 2 * pl.chains * (pl.nseg - 1));
    auto go = [&](auto tag) {
        using T = decltype(tag);
        if (a->dk <= 64) return vec ? run<T, 64, true>(p, pl, a->nb, redo, stream) : run<T, 64, false>(p, pl, a->nb, redo, stream);
        return vec ? run<T, 128, true>(p, pl, a->nb, redo, stream) : run<T, 128, false>(p, pl, a->nb, redo, stream);
    };
    const int rc = a->dtype == NEED_F32 ? go(float{}) : a->dtype == NEED_BF16 ? go(__nv_bfloat16{}) : go(__half{});
    return rc != NEED_OK ? rc : ok();
}

}  // extern "C"
