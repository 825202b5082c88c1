// token_log_probs.cu -- log probabilities of given tokens, the entropy and the largest
// alternatives of rows of logits (need_token_log_probs), and the gradient
// (need_token_log_probs_backward).  With x = logits / temperature, m its largest,
//
//   S = sum e^{x - m},  log p_j = x_j - m - log S,  H = log S - sum e^{x - m} (x - m) / S
//   dx_j = g (1[j = token] - p_j) - gh p_j (log p_j + H)
//
// The sums run in one pass with a running maximum, which a warp shares; what they leave
// out are the maxima themselves, which are counted: with r the rest, log S = log(count) +
// log1p(r / count), so that probabilities near 1 and small entropies keep their relative
// precision (both terms of H are positive).
//
// The largest: the k-th of the lanes' maxima is a bound that k logits reach.  The first pass
// leaves the maxima of a thread's pieces, some 32 logits each; only those that reach the
// bound are read again, and what they hold is put into order by counting.  Keys order by
// value, then by the lower token.
//
// Short rows take a warp each, longer ones a block of 4; where there are few, rows are cut
// into parts that a second launch joins, in order.  Rows of any alignment: the elements before
// the first and after the last whole 16 bytes are taken one by one.  Per logit: 2 or 4 B, one
// ex2 (16 a cycle and SM, three quarters of HBM's time for 16 bits) and some 7 other
// instructions, half of them in packed pairs.  1024 rows of 50021 bf16 logits: 24 us (4.3
// TB/s), with the 20 largest 31.6 -- all rows run side by side, so that what follows the
// pass, some 7 us of waiting on one another, hides under nothing; fp32 34.6 us (5.9 TB/s).
// 16384 rows of 784: 10 us, the gradient 14.  4 rows of 131072 fp32 logits, the 5 largest: 9
// us, two launches.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <float.h>

#include <algorithm>
#include <type_traits>

#include "host_common.h"
#include "need_scan.h"

using namespace need;

namespace {

constexpr int kThreads = 128, kWarps = kThreads / 32;
constexpr int kJoin = 256, kMaxParts = kJoin;  // a lane each
constexpr int UN = 4;              // 16-byte pieces of a lane in flight
constexpr int kList = 512;         // keys that a block gathers (a warp of its own: a quarter)
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.69314718055994531f;
constexpr float kLow = -200.0f;    // 2^kLow is 0, and its product with kLow too
constexpr int kGroups = 16;
constexpr int kNone = static_cast<int>(0x80000000u);  // below order(-infinity)
using u64 = unsigned long long;

struct LogpParams {
    const void* logits;
    int64_t stride;
    const int64_t* tokens;
    float* log_prob;
    float* entropy;
    float* stats;
    float* top_lp;
    int64_t* top_id;
    int64_t rows, V, len;  // len: logits of a part
    int32_t top, parts;
    float inv_t;
    float4* part;          // [rows, parts]: m, count, r, u
    u64* part_top;         // [rows, parts, top]
    const float* g;
    const float* gh;
    void* grad;
    int64_t grad_stride;
};

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float nan32() { return __int_as_float(0x7fc00000); }

template <typename T>
struct Vec {
    static constexpr int N = 16 / sizeof(T);
    static __device__ __forceinline__ void widen(const uint4& u, float* f) {
        if constexpr (std::is_same<T, __nv_bfloat16>::value) {  // a shift and a mask
            const uint32_t* w = reinterpret_cast<const uint32_t*>(&u);
#pragma unroll
            for (int i = 0; i < N; i += 2) f[i] = __uint_as_float(w[i / 2] << 16), f[i + 1] = __uint_as_float(w[i / 2] & 0xffff0000u);
        } else {
            const T* e = reinterpret_cast<const T*>(&u);
#pragma unroll
            for (int i = 0; i < N; ++i) f[i] = to_float(e[i]);
        }
    }
};

// The largest of 16-byte pieces (a NaN is none).
template <int K>
__device__ __forceinline__ float most(const uint4 (&u)[K], float) {
    float m = -INFINITY;
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const float* x = reinterpret_cast<const float*>(&u[k]);
        m = fmaxf(m, fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])));
    }
    return m;
}
template <typename T2, int K>
__device__ __forceinline__ float most_of_pairs(const uint4 (&u)[K]) {
    const T2* x = reinterpret_cast<const T2*>(&u[0]);
    T2 m = x[0];
#pragma unroll
    for (int i = 1; i < 4 * K; ++i) m = __hmax2(m, x[i]);
    return fmaxf(fmaxf(to_float(m.x), to_float(m.y)), -INFINITY);
}
template <int K>
__device__ __forceinline__ float most(const uint4 (&u)[K], __nv_bfloat16) { return most_of_pairs<__nv_bfloat162>(u); }
template <int K>
__device__ __forceinline__ float most(const uint4 (&u)[K], __half) { return most_of_pairs<__half2>(u); }
// A piece of -infinity.
__device__ __forceinline__ uint4 lowest(float) { return make_uint4(0xff800000u, 0xff800000u, 0xff800000u, 0xff800000u); }
__device__ __forceinline__ uint4 lowest(__nv_bfloat16) { return make_uint4(0xff80ff80u, 0xff80ff80u, 0xff80ff80u, 0xff80ff80u); }
__device__ __forceinline__ uint4 lowest(__half) { return make_uint4(0xfc00fc00u, 0xfc00fc00u, 0xfc00fc00u, 0xfc00fc00u); }
// How many of a piece are m; -infinity in their places.
__device__ __forceinline__ float take(uint4& u, float m, float) {
    float n = 0.0f, *x = reinterpret_cast<float*>(&u);
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (x[i] == m) n += 1.0f, x[i] = -INFINITY;
    return n;
}
template <typename T2>
__device__ __forceinline__ float take_of_pairs(uint4& u, T2 m, uint32_t low) {
    int n = 0;
    uint32_t* x = reinterpret_cast<uint32_t*>(&u);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t is = __heq2_mask(reinterpret_cast<const T2*>(&u)[i], m);
        n += __popc(is);
        x[i] = (x[i] & ~is) | (low & is);
    }
    return static_cast<float>(n >> 4);
}
__device__ __forceinline__ float take(uint4& u, float m, __nv_bfloat16) { return take_of_pairs(u, __float2bfloat162_rn(m), 0xff80ff80u); }
__device__ __forceinline__ float take(uint4& u, float m, __half) { return take_of_pairs(u, __float2half2_rn(m), 0xfc00fc00u); }

// A run of a row's logits: `head` elements, `nvec` whole 16-byte pieces, `tail` elements.
template <typename T>
struct Run {
    static constexpr int N = Vec<T>::N;
    const T* x;
    int nvec, head, tail;
    __device__ __forceinline__ Run(const T* x_, int64_t len) : x(x_) {
        const int off = static_cast<int>((reinterpret_cast<uintptr_t>(x_) & 15u) / sizeof(T));
        const int64_t h = off == 0 ? 0 : N - off;
        head = static_cast<int>(h < len ? h : len);
        nvec = static_cast<int>((len - head) / N);
        tail = static_cast<int>(len - head) - nvec * N;
    }
    __device__ __forceinline__ const uint4* body() const { return reinterpret_cast<const uint4*>(x + head); }
    __device__ __forceinline__ int edges() const { return head + tail; }
    __device__ __forceinline__ int edge(int n) const { return n < head ? n : nvec * N + n; }  // its index
};

// ------------------------------------------------------------------ sums
struct Sums {
    float m, cnt, r, u;  // the largest, how many equal it, the others' sum of 2^z, and of z 2^z
};
// b joined to a
__device__ __forceinline__ void join(Sums& a, const Sums& b, float c) {
    const float m = fmaxf(a.m, b.m);
    const float da = a.m == m ? 0.0f : fmaxf((a.m - m) * c, kLow), db = b.m == m ? 0.0f : fmaxf((b.m - m) * c, kLow);
    const float fa = a.m == m ? 1.0f : ex2(da), fb = b.m == m ? 1.0f : ex2(db);
    // of a side below the maximum the largest are among the rest
    const float ra = a.m == m ? a.r : fa * (a.r + a.cnt), rb = b.m == m ? b.r : fb * (b.r + b.cnt);
    a.u = fa * (a.u + da * (a.r + a.cnt)) + fb * (b.u + db * (b.r + b.cnt));
    a.cnt = (a.m == m ? a.cnt : 0.0f) + (b.m == m ? b.cnt : 0.0f);
    a.r = ra + rb;
    a.m = m;
}
__device__ __forceinline__ int order(float x) {  // signed, no NaN
    const int b = __float_as_int(x);
    return b ^ ((b >> 31) & 0x7fffffff);
}
__device__ __forceinline__ float unorder(int k) { return __int_as_float(k ^ ((k >> 31) & 0x7fffffff)); }

// The warp's largest logit raised to lm, the largest of those to come (s.m is the warp's,
// the rest the lane's); whether the largest are among these.
__device__ __forceinline__ bool raise(float lm, Sums& s, float c) {
    const float wm = unorder(__reduce_max_sync(0xffffffffu, order(lm)));
    if (wm > s.m) {
        const float d = fmaxf((s.m - wm) * c, kLow), f = ex2(d);
        s.u = f * (s.u + d * (s.r + s.cnt));
        s.r = f * (s.r + s.cnt);
        s.cnt = 0.0f, s.m = wm;
    }
    return wm == s.m && wm > -INFINITY;
}
// K logits of a lane (none above m, none that is the largest) into sums of pairs.
template <int K>
__device__ __forceinline__ void add(const float (&x)[K], float m, float c, float2& r, float2& u) {
    const float2 mm = make_float2(-m, -m), cc = make_float2(c, c);
#pragma unroll
    for (int i = 0; i < K; i += 2) {
        const float2 z = __fmul2_rn(__fadd2_rn(make_float2(x[i], x[i + 1]), mm), cc), e = make_float2(ex2(z.x), ex2(z.y));
        r = __fadd2_rn(r, e);
        u = __ffma2_rn(e, make_float2(fmaxf(z.x, kLow), fmaxf(z.y, kLow)), u);
    }
}

// ------------------------------------------------------------------ keys
__device__ __forceinline__ u64 key_of(float x, int64_t i) {
    const uint32_t v = x != x ? 0xffffffffu : static_cast<uint32_t>(order(x + 0.0f)) ^ 0x80000000u;  // -0 as 0
    return (static_cast<u64>(v) << 32) | (0xffffffffu - static_cast<uint32_t>(i));
}
__device__ __forceinline__ float value_of(u64 k) {
    const uint32_t v = static_cast<uint32_t>(k >> 32);
    return v == 0xffffffffu ? nan32() : unorder(static_cast<int>(v ^ 0x80000000u));
}
__device__ __forceinline__ int64_t token_of(u64 k) { return 0xffffffffu - static_cast<uint32_t>(k); }

// The `top` largest of n keys in order, 0 behind them; threads t, t + step, ...
__device__ __forceinline__ void rank_keys(const u64* keys, int n, int top, u64* out, int t, int step) {
    for (int i = t; i < n; i += step) {
        const u64 k = keys[i];
        int r = 0;
        if (k == 0) continue;
        for (int j = 0; j < n; ++j) r += keys[j] > k ? 1 : 0;
        if (r < top) out[r] = k;
    }
}
// The `top` largest of a warp's lists, in order themselves, one a lane.
__device__ __forceinline__ void merge(const u64* list, int n, int top, u64* out, int lane) {
    int at = 0;
    u64 k = n > 0 ? list[0] : 0;
    for (int i = 0; i < top; ++i) {
        const uint32_t hi = __reduce_max_sync(0xffffffffu, static_cast<uint32_t>(k >> 32));
        const uint32_t lo = __reduce_max_sync(0xffffffffu, static_cast<uint32_t>(k >> 32) == hi ? static_cast<uint32_t>(k) : 0u);
        const u64 best = (static_cast<u64>(hi) << 32) | lo;
        if (lane == 0) out[i] = best;
        if (k == best && k != 0) k = ++at < n ? list[at] : 0;  // one lane's: keys differ
    }
}

// ------------------------------------------------------------------ the row's results
struct Result {
    float m, l, inv_t;  // the largest logit, log S
    __device__ __forceinline__ float log_p(float x) const { return m == -INFINITY ? l - INFINITY : fmaf(x - m, inv_t, -l); }
};
// The logit of the row's token.
template <typename T>
__device__ __forceinline__ float given(const LogpParams& p, int64_t row, int64_t tok) {
    return tok >= 0 && tok < p.V ? to_float(static_cast<const T*>(p.logits)[row * p.stride + tok]) : 0.0f;
}
// One thread writes the row's log p (tok the token, x its logit), entropy and stats.
__device__ __forceinline__ Result finish(const LogpParams& p, int64_t row, const Sums& s, bool write, int64_t tok, float x) {
    Result res{s.m, 0.0f, p.inv_t};
    float h = 0.0f;
    if (s.m == INFINITY || s.r != s.r) {
        res.l = h = nan32();
    } else if (s.m > -INFINITY) {
        res.l = s.cnt == 1.0f ? log1pf(s.r) : logf(s.cnt) + log1pf(s.r / s.cnt);
        h = res.l - kLn2 * (s.u / (s.cnt + s.r));
    }
    if (write) {
        float lp = 0.0f;
        if (tok >= p.V) lp = nan32();
        else if (tok >= 0) lp = res.log_p(x);
        p.log_prob[row] = lp, p.entropy[row] = h;
        if (p.stats != nullptr) p.stats[2 * row] = s.m, p.stats[2 * row + 1] = res.l;
    }
    return res;
}
__device__ __forceinline__ void write_top(const LogpParams& p, int64_t row, const Result& res, const u64* keys, int t, int step) {
    for (int i = t; i < p.top; i += step) {
        const u64 k = keys[i];
        p.top_lp[row * p.top + i] = k == 0 ? (res.l != res.l ? res.l : -INFINITY) : res.log_p(value_of(k));
        p.top_id[row * p.top + i] = k == 0 ? -1 : token_of(k);
    }
}

// ------------------------------------------------------------------ kernels
// WPR warps a row: 1, or all of the block's, which then take part blockIdx.y of the row.
template <typename T, int WPR>
__global__ void __launch_bounds__(kThreads) logp_kernel(const LogpParams p) {
    constexpr int N = Vec<T>::N, TEAM = 32 * WPR, CAP = kList * WPR / kWarps;
    __shared__ Sums s_sums[kWarps];
    __shared__ float s_best[kGroups][kThreads];  // the largest of a thread's pieces, a group of batches each
    __shared__ int s_max[kWarps * (NEED_TOKEN_LOG_PROBS_MAX_TOP + 1) / 2], s_low;
    __shared__ u64 s_keys[kList], s_top[kWarps * NEED_TOKEN_LOG_PROBS_MAX_TOP];
    __shared__ int s_n[kWarps];
    auto sync = [] {
        if (WPR == 1) __syncwarp();
        else __syncthreads();
    };
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int team = warp / WPR, tt = threadIdx.x % TEAM;
    const int64_t row = int64_t(blockIdx.x) * (kWarps / WPR) + team;
    if (row >= p.rows) return;  // a whole team
    const int64_t first = int64_t(blockIdx.y) * p.len;
    const Run<T> run(static_cast<const T*>(p.logits) + row * p.stride + first, p.len < p.V - first ? p.len : p.V - first);
    const float c = p.inv_t * kLog2e;

    const int64_t tok = tt == 0 ? p.tokens[row] : -1;
    const float xt = given<T>(p, row, tok);
    Sums s{-INFINITY, 0.0f, 0.0f, 0.0f};
    float tm = -INFINITY, best = -INFINITY;
    const int batches = (run.nvec + TEAM * UN - 1) / (TEAM * UN), size = (batches + kGroups - 1) / kGroups;
    int group = 0, left = size;
    // the pieces, UN a lane at a time; every lane of a warp takes part in every batch
    auto load = [&](uint4 (&u)[UN], int v0) {
        if (v0 + TEAM * UN <= run.nvec) {
#pragma unroll
            for (int k = 0; k < UN; ++k) u[k] = __ldg(run.body() + v0 + k * TEAM + tt);
        } else {
#pragma unroll
            for (int k = 0; k < UN; ++k) u[k] = v0 + k * TEAM + tt < run.nvec ? __ldg(run.body() + v0 + k * TEAM + tt) : lowest(T{});
        }
    };
    auto batch = [&](uint4 (&u)[UN], int v0) {
        const float lm = most(u, T{});
        if (raise(lm, s, c)) {
#pragma unroll
            for (int k = 0; k < UN; ++k) {
                const uint4 w[1] = {u[k]};
                if (__any_sync(0xffffffffu, most(w, T{}) == s.m)) s.cnt += take(u[k], s.m, T{});
            }
        }
        const float m = s.m == -INFINITY ? 0.0f : s.m;
        float2 sr = make_float2(0.0f, 0.0f), su = sr;
#pragma unroll
        for (int k = 0; k < UN; ++k) {
            if (v0 + k * TEAM + (tt & ~31) >= run.nvec) break;
            float x[N];
            Vec<T>::widen(u[k], x);
            add(x, m, c, sr, su);
        }
        s.r += sr.x + sr.y, s.u += su.x + su.y;
        best = fmaxf(best, lm);
        if (p.top > 0 && (--left == 0 || v0 + TEAM * UN >= run.nvec)) {
            s_best[group][threadIdx.x] = s.r == s.r ? best : INFINITY;  // there may be a NaN in it
            tm = fmaxf(tm, best);
            best = -INFINITY, left = size, ++group;
        }
    };
    if constexpr (WPR == 1) {
        for (int v0 = 0; v0 < run.nvec; v0 += TEAM * UN) {
            uint4 u[UN];
            load(u, v0);
            batch(u, v0);
        }
    } else {  // the next ones on their way meanwhile
        uint4 u[UN], w[UN];
        load(u, 0);
        for (int v0 = 0; v0 < run.nvec; v0 += 2 * TEAM * UN) {
            if (v0 + TEAM * UN < run.nvec) load(w, v0 + TEAM * UN);
            batch(u, v0);
            if (v0 + TEAM * UN >= run.nvec) break;
            if (v0 + 2 * TEAM * UN < run.nvec) load(u, v0 + 2 * TEAM * UN);
            batch(w, v0 + TEAM * UN);
        }
    }
    if (warp % WPR == 0 && run.edges() > 0) {
        float x[2] = {lane < run.edges() ? to_float(run.x[run.edge(lane)]) : -INFINITY, -INFINITY};
        const float lm = fmaxf(x[0], -INFINITY);
        if (raise(lm, s, c) && x[0] == s.m) s.cnt += 1.0f, x[0] = -INFINITY;
        float2 sr = make_float2(0.0f, 0.0f), su = sr;
        add(x, s.m == -INFINITY ? 0.0f : s.m, c, sr, su);
        s.r += sr.x, s.u += su.x;
        tm = fmaxf(tm, lm);
    }
#pragma unroll
    for (int m = 16; m >= 1; m >>= 1) {
        s.cnt += __shfl_xor_sync(0xffffffffu, s.cnt, m);
        s.r += __shfl_xor_sync(0xffffffffu, s.r, m);
        s.u += __shfl_xor_sync(0xffffffffu, s.u, m);
    }
    if (WPR > 1) {
        if (lane == 0) s_sums[warp] = s;
        __syncthreads();
        s = s_sums[0];
        for (int w = 1; w < WPR; ++w) join(s, s_sums[w], c);
    }

    u64* const keys = s_keys + team * CAP;
    u64* const top = s_top + team * NEED_TOKEN_LOG_PROBS_MAX_TOP;
    if (p.top > 0) {
        // a bound that `top` logits reach: of the lanes' largest the top-th, or, of several
        // warps, the top-th of the (top + 1) / 2 that each hands in
        if (tt == 0) s_n[team] = 0;
        for (int i = tt; i < p.top; i += TEAM) top[i] = 0;
        const int give = WPR == 1 ? p.top : (p.top + 1) / 2;
        int v = order(tm), at = v;
        for (int i = 0; i < give; ++i) {
            at = __reduce_max_sync(0xffffffffu, v);
            if (lane == __ffs(__ballot_sync(0xffffffffu, v == at)) - 1) {
                v = kNone;
                if (WPR > 1) s_max[warp * give + i] = at;
            }
        }
        if (WPR > 1) {
            // equal values in order of their places, so that one is the top-th
            __syncthreads();
            if (tt < WPR * give) {
                const int mine = s_max[tt];
                int above = 0;
                for (int i = 0; i < WPR * give; ++i) above += s_max[i] > mine || (s_max[i] == mine && i < tt) ? 1 : 0;
                if (above == p.top - 1) s_low = mine;
            }
            __syncthreads();
            at = s_low;
        }
        sync();
        const float low = unorder(at), thr = low > -FLT_MAX ? low : -FLT_MAX;
        auto gather = [&](int i) {
            const float x = to_float(run.x[i]);
            if (!(x < thr)) {
                const int n = atomicAdd(&s_n[team], 1);
                if (n < CAP) keys[n] = key_of(x, first + i);
            }
        };
        auto each = [&](auto&& f) {
            for (int v = tt; v < run.nvec; v += TEAM) {
                float x[N];
                Vec<T>::widen(__ldg(run.body() + v), x);
#pragma unroll
                for (int e = 0; e < N; ++e) f(x[e], run.head + v * N + e);
            }
            if (tt < run.edges()) f(to_float(run.x[run.edge(tt)]), run.edge(tt));
        };
        const bool ordered = s.r == s.r;  // no NaN
        unsigned hit = 0;
        for (int g = 0; g < group; ++g) hit |= (s_best[g][threadIdx.x] < thr ? 0u : 1u) << g;
        for (; hit != 0; hit &= hit - 1) {
            const int b0 = (__ffs(hit) - 1) * size;
            for (int b = b0; b < b0 + size && b < batches; ++b) {
                const int v0 = b * (TEAM * UN) + tt;
                uint4 u[UN];
#pragma unroll
                for (int k = 0; k < UN; ++k) u[k] = v0 + k * TEAM < run.nvec ? __ldg(run.body() + v0 + k * TEAM) : lowest(T{});
                unsigned pieces = 0;
#pragma unroll
                for (int k = 0; k < UN; ++k) {
                    const uint4 w[1] = {u[k]};
                    if (v0 + k * TEAM < run.nvec && !(ordered && most(w, T{}) < thr)) pieces |= 1u << k;
                }
                for (; pieces != 0; pieces &= pieces - 1) {
                    const int v = v0 + (__ffs(pieces) - 1) * TEAM;
                    float x[N];
                    Vec<T>::widen(__ldg(run.body() + v), x);
                    unsigned elements = 0;
#pragma unroll
                    for (int e = 0; e < N; ++e) elements |= (x[e] < thr ? 0u : 1u) << e;
                    for (; elements != 0; elements &= elements - 1) gather(run.head + v * N + __ffs(elements) - 1);
                }
            }
        }
        if (tt < run.edges()) gather(run.edge(tt));
        sync();
        const int n = s_n[team];
        if (n <= CAP) {
            rank_keys(keys, n, p.top, top, tt, TEAM);
        } else {  // too many reach the bound: one after another, a pass each
            u64 below = ~0ull;
            for (int k = 0; k < p.top; ++k) {
                u64 best = 0;
                each([&](float x, int i) {
                    const u64 key = x == -INFINITY ? 0 : key_of(x, first + i);
                    if ((k == 0 || key < below) && key > best) best = key;  // a NaN at token 0 has the largest key there is
                });
#pragma unroll
                for (int m = 16; m >= 1; m >>= 1) {
                    const u64 o = __shfl_xor_sync(0xffffffffu, best, m);
                    best = o > best ? o : best;
                }
                if (WPR > 1) {
                    __syncthreads();  // the keys of the last round have been read
                    if (lane == 0) s_keys[warp] = best;
                    __syncthreads();
                    for (int w = 0; w < WPR; ++w) best = s_keys[w] > best ? s_keys[w] : best;
                }
                if (tt == 0) top[k] = best;
                if (best == 0) break;
                below = best;
            }
        }
        sync();
    }
    if (p.parts > 1) {
        const int64_t at = row * p.parts + blockIdx.y;
        if (tt == 0) p.part[at] = make_float4(s.m, s.cnt, s.r, s.u);
        for (int i = tt; i < p.top; i += TEAM) p.part_top[at * p.top + i] = top[i];
        return;
    }
    const Result res = finish(p, row, s, tt == 0, tok, xt);
    if (p.top > 0) write_top(p, row, res, top, tt, TEAM);
}

// A block joins a row's parts, a lane each.
template <typename T>
__global__ void __launch_bounds__(kJoin) join_kernel(const LogpParams p) {
    constexpr int MT = NEED_TOKEN_LOG_PROBS_MAX_TOP, W = kJoin / 32;
    __shared__ u64 s_lists[W * MT], s_top[MT];
    __shared__ Sums s_sums[W];
    const int64_t row = blockIdx.x;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const bool have = threadIdx.x < p.parts;
    const float c = p.inv_t * kLog2e;
    const int64_t at = row * p.parts + threadIdx.x, tok = p.tokens[row];
    const float xt = given<T>(p, row, tok);
    Sums s{-INFINITY, 0.0f, 0.0f, 0.0f};
    if (have) {
        const float4 f = p.part[at];
        s = Sums{f.x, f.y, f.z, f.w};
    }
#pragma unroll
    for (int m = 1; m <= 16; m <<= 1) {
        const Sums o{__shfl_xor_sync(0xffffffffu, s.m, m), __shfl_xor_sync(0xffffffffu, s.cnt, m), __shfl_xor_sync(0xffffffffu, s.r, m),
                     __shfl_xor_sync(0xffffffffu, s.u, m)};
        join(s, o, c);
    }
    if (lane == 0) s_sums[warp] = s;
    if (p.top > 0) merge(p.part_top + at * p.top, have ? p.top : 0, p.top, s_lists + warp * MT, lane);
    __syncthreads();
    if (warp > 0) return;
    for (int w = 1; w < W; ++w) join(s, s_sums[w], c);
    if (p.top > 0) merge(s_lists + lane * MT, lane < W ? p.top : 0, p.top, s_top, lane);
    __syncwarp();
    const Result res = finish(p, row, s, lane == 0, tok, xt);
    if (p.top > 0) write_top(p, row, res, s_top, lane, 32);
}

// A warp takes 32 * UN pieces of a row.  SAME: the gradient's rows lie as the logits' do
// within 16 bytes.  The token's own place is written again, by 1 - p from log p, since p may
// be near 1.
template <typename T, bool SAME>
__global__ void __launch_bounds__(kThreads) logp_backward_kernel(const LogpParams p) {
    constexpr int N = Vec<T>::N;
    const int lane = threadIdx.x & 31;
    const int64_t id = int64_t(blockIdx.x) * kWarps + (threadIdx.x >> 5), row = id / p.parts;
    const int part = static_cast<int>(id % p.parts);
    if (row >= p.rows) return;
    const Run<T> run(static_cast<const T*>(p.logits) + row * p.stride, p.V);
    T* const out = static_cast<T*>(p.grad) + row * p.grad_stride;
    uint4 u[UN];
    const int v0 = part * 32 * UN + lane;
#pragma unroll
    for (int k = 0; k < UN; ++k)
        if (v0 + k * 32 < run.nvec) u[k] = __ldcs(run.body() + v0 + k * 32);
    const float m = p.stats[2 * row], l = p.stats[2 * row + 1], h = p.entropy[row];
    const float g = p.g != nullptr ? p.g[row] : 0.0f, gh = p.gh != nullptr ? p.gh[row] : 0.0f;
    const int64_t tok = p.tokens[row];
    const float gt = tok >= p.V ? nan32() : tok >= 0 ? g : 0.0f;  // of the token's log p
    const bool none = m == -INFINITY && l == l;                   // a row of nothing
    const float c = p.inv_t * kLog2e, ms = none ? 0.0f : m;
    const float a = p.inv_t * -(gt + gh * h), b = p.inv_t * -gh * kLn2;  // dx = p (a + b log2 p)
    const float2 mm = make_float2(-ms, -ms), cc = make_float2(c, c), ll = make_float2(-l * kLog2e, -l * kLog2e);
    const float2 aa = make_float2(a, a), bb = make_float2(b, b);
    auto grad = [&](float x, float y) {
        const float2 z = __ffma2_rn(__fadd2_rn(make_float2(x, y), mm), cc, ll);
        return __fmul2_rn(make_float2(ex2(z.x), ex2(z.y)), __ffma2_rn(bb, make_float2(fmaxf(z.x, kLow), fmaxf(z.y, kLow)), aa));
    };
    const float zero = gt == gt ? 0.0f : gt;  // a row of nothing's gradient
#pragma unroll
    for (int k = 0; k < UN; ++k) {
        const int v = v0 + k * 32;
        if (v >= run.nvec) break;
        const int64_t i0 = run.head + int64_t(v) * N;
        float x[N];
        Vec<T>::widen(u[k], x);
        union { uint4 u; T e[N]; } r;
#pragma unroll
        for (int e = 0; e < N; e += 2) {
            const float2 d = none ? make_float2(zero, zero) : grad(x[e], x[e + 1]);
            r.e[e] = static_cast<T>(d.x), r.e[e + 1] = static_cast<T>(d.y);
        }
        if constexpr (SAME) {
            __stcs(reinterpret_cast<uint4*>(out + i0), r.u);
        } else {
#pragma unroll
            for (int e = 0; e < N; ++e) out[i0 + e] = r.e[e];
        }
    }
    if (part == 0 && lane < run.edges()) {
        const int i = run.edge(lane);
        out[i] = static_cast<T>(none ? zero : grad(to_float(run.x[i]), 0.0f).x);
    }
    if (none || tok < 0 || tok >= p.V) return;
    // after the stores above, by the thread that made the one at its place
    const int64_t in = tok - run.head;
    const bool body = in >= 0 && in < int64_t(run.nvec) * N;
    const int v = static_cast<int>(in / N);
    const bool mine = body ? v / (32 * UN) == part && (v & 31) == lane : part == 0 && lane == (in < 0 ? tok : tok - int64_t(run.nvec) * N);
    if (mine) {
        const float lp = fmaf(to_float(run.x[tok]) - ms, p.inv_t, -l);
        const float q = expf(lp);
        out[tok] = static_cast<T>(p.inv_t * (gt * -expm1f(lp) - gh * q * (fmaxf(lp, kLow) + h)));
    }
}

// ------------------------------------------------------------------ host
// A warp's lanes give a bound for few alternatives only: of 4096 rows of 784 bf16 logits
// the 5 largest take it 8.6 us and a block 20, but the 32 largest 125 and 31.  V: without
// alternatives 4096 rows of 2048 take a warp 6.9 us each and a block 9.4.
// Cut: 150 rows of 131072 fp32 logits go from 50 us (uncut) to 16.5; below 4 batches, and
// for more rows below 16, the join costs more (300 rows of 16384 bf16 logits: 7.8 us in two
// parts, 6.4 uncut; 500 of 131072 fp32: 51 and 67).
struct Shape {
    bool wide;      // a block a row or part
    int32_t parts;
    int64_t len;
};
Shape shape_of(int32_t dtype, int64_t rows, int64_t V, int32_t top) {
    const int n = 16 / dtype_bytes(dtype);
    Shape s{V > 2048 || top > 16, 1, V};
    const int64_t batch = int64_t(kThreads) * UN * n, batches = (V + batch - 1) / batch, places = batches < 16 ? 296 : 592;
    if (s.wide && batches >= 4 && rows < places) {
        const int64_t parts = std::min({(places + rows - 1) / rows, batches, int64_t(kMaxParts)});
        s.len = (V + parts - 1) / parts;
        s.len = (s.len + n - 1) / n * n;  // parts lie alike within 16 bytes
        s.parts = int32_t((V + s.len - 1) / s.len);
    }
    return s;
}

int check_args(const need_token_log_probs_args* a) {
    if (a == nullptr) return fail(NEED_ERR_INVALID, "token log probs: args is null");
    if (!dtype_ok(a->dtype)) return fail(NEED_ERR_UNSUPPORTED, "token log probs: dtype %d", a->dtype);
    if (a->rows < 1 || a->V < 1) return fail(NEED_ERR_INVALID, "token log probs: sizes must be positive");
    if (a->rows > (int64_t(1) << 31) - 1 || a->V > (int64_t(1) << 31) - 1)
        return fail(NEED_ERR_UNSUPPORTED, "token log probs: at most 2^31 - 1 rows and logits a row");
    if (a->logits == nullptr || a->tokens == nullptr || a->entropy == nullptr)
        return fail(NEED_ERR_INVALID, "token log probs: logits, tokens and entropy are required");
    if (!(a->temperature >= 1e-30 && a->temperature <= 1e30)) return fail(NEED_ERR_INVALID, "token log probs: temperature must lie in [1e-30, 1e30]");
    return NEED_OK;
}
LogpParams params(const need_token_log_probs_args* a) {
    LogpParams p{};
    p.logits = a->logits, p.stride = a->stride, p.tokens = a->tokens, p.log_prob = a->log_prob, p.entropy = a->entropy;
    p.stats = a->stats, p.rows = a->rows, p.V = a->V, p.inv_t = static_cast<float>(1.0 / a->temperature);
    return p;
}

}  // namespace

extern "C" {

size_t need_token_log_probs_workspace_size(int32_t dtype, int64_t rows, int64_t V, int32_t top) {
    if (!dtype_ok(dtype) || rows < 1 || V < 1 || top < 0) return 16;
    const Shape s = shape_of(dtype, rows, V, top);
    return s.parts == 1 ? 16 : size_t(rows) * s.parts * (sizeof(float4) + sizeof(u64) * top);
}

int need_token_log_probs(const need_token_log_probs_args* a, need_stream_t stream) {
    int rc = check_args(a);
    if (rc != NEED_OK) return rc;
    if (a->log_prob == nullptr) return fail(NEED_ERR_INVALID, "token log probs: log_prob is required");
    if (a->top < 0 || a->top > a->V || (a->top > 0 && (a->top_log_probs == nullptr || a->top_tokens == nullptr)))
        return fail(NEED_ERR_INVALID, "token log probs: 0 to V alternatives, and their outputs");
    if (a->top > NEED_TOKEN_LOG_PROBS_MAX_TOP)
        return fail(NEED_ERR_UNSUPPORTED, "token log probs: at most %d alternatives", NEED_TOKEN_LOG_PROBS_MAX_TOP);
    const Shape s = shape_of(a->dtype, a->rows, a->V, a->top);
    if (s.parts > 1 && (a->workspace == nullptr || !aligned16(a->workspace) ||
                        a->workspace_bytes < need_token_log_probs_workspace_size(a->dtype, a->rows, a->V, a->top)))
        return fail(NEED_ERR_WORKSPACE, "token log probs: workspace missing, misaligned or too small");
    LogpParams p = params(a);
    p.top = a->top, p.top_lp = a->top_log_probs, p.top_id = a->top_tokens, p.parts = s.parts, p.len = s.len;
    if (s.parts > 1) {
        p.part = static_cast<float4*>(a->workspace);
        p.part_top = reinterpret_cast<u64*>(p.part + a->rows * s.parts);
    }
    auto run = [&](auto tag) {
        using T = decltype(tag);
        if (s.wide) logp_kernel<T, kWarps><<<dim3(static_cast<unsigned>(a->rows), s.parts), kThreads, 0, stream>>>(p);
        else logp_kernel<T, 1><<<static_cast<unsigned>((a->rows + kWarps - 1) / kWarps), kThreads, 0, stream>>>(p);
        if (s.parts > 1) join_kernel<T><<<static_cast<unsigned>(a->rows), kJoin, 0, stream>>>(p);
    };
    if (a->dtype == NEED_F32) run(float{});
    else if (a->dtype == NEED_BF16) run(__nv_bfloat16{});
    else run(__half{});
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? ok() : cuda_fail(e, "token log probs launch");
}

int need_token_log_probs_backward(const need_token_log_probs_args* a, need_stream_t stream) {
    int rc = check_args(a);
    if (rc != NEED_OK) return rc;
    if (a->stats == nullptr || a->grad == nullptr) return fail(NEED_ERR_INVALID, "token log probs: stats and grad are required");
    if (a->rows > 1 && a->grad_stride < a->V) return fail(NEED_ERR_INVALID, "token log probs: the gradient's rows overlap");
    LogpParams p = params(a);
    const int es = dtype_bytes(a->dtype), n = 16 / es;
    const int64_t parts = std::max<int64_t>(1, (a->V / n + 32 * UN - 1) / (32 * UN)), blocks = (a->rows * parts + kWarps - 1) / kWarps;
    if (blocks > (int64_t(1) << 31) - 1) return fail(NEED_ERR_UNSUPPORTED, "token log probs: too many logits");
    p.parts = static_cast<int32_t>(parts), p.g = a->g_log_prob, p.gh = a->g_entropy, p.grad = a->grad, p.grad_stride = a->grad_stride;
    const bool same = (reinterpret_cast<uintptr_t>(a->logits) - reinterpret_cast<uintptr_t>(a->grad)) % 16 == 0 &&
                      (a->rows == 1 || (a->stride - a->grad_stride) * es % 16 == 0);
    auto run = [&](auto tag) {
        using T = decltype(tag);
        if (same) logp_backward_kernel<T, true><<<static_cast<unsigned>(blocks), kThreads, 0, stream>>>(p);
        else logp_backward_kernel<T, false><<<static_cast<unsigned>(blocks), kThreads, 0, stream>>>(p);
    };
    if (a->dtype == NEED_F32) run(float{});
    else if (a->dtype == NEED_BF16) run(__nv_bfloat16{});
    else run(__half{});
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? ok() : cuda_fail(e, "token log probs launch");
}

}  // extern "C"
