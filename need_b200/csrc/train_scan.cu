// train_scan.cu -- the gated and SSD recurrences for training: a forward that
// keeps what its backward needs, and the backward (need_scan_train_forward,
// need_scan_train_backward).
//
//   GATED  a = s(z), w = s(g) x
//   SSD    a = exp(-(dt_min + dt_scale s(dt))), w = s(bg) u
//   h_t = [t starts a segment ? 0 : a_t h_{t-1}] + (1 - a_t) w_t
//   GATED  out = h          SSD  out = (s(cg) h + D u) s(og)
//
// With e_t the gradient reaching h_t from out (GATED: gout; SSD: gout s(og)
// s(cg)) and mu_T the gradient of the final state, the backward runs
//   lam_t = e_t + mu_{t+1},   mu_t = [t starts a segment ? 0 : a_t lam_t]
// from the last token to the first.  Written for mu, the recurrence uses each
// row's own a_t, so a tile needs no row of its neighbour.  Then
//   d a_t = lam_t ([start ? 0 : h_{t-1}] - w_t),  d w_t = lam_t (1 - a_t),
// the gates' own derivatives, and grad_h0 = mu_0.
//
// Precision: gates, states and gradients in fp32, rounded once to the stream's
// dtype on the way out (the forward-only scans of scan_kernel.cuh round every
// gate op as the reference's torch path does; a gradient of those roundings
// would be the gradient of another function).  1 - s(x) is formed from the
// exponential, not by subtraction, so it keeps its relative precision.
//
// A reset is a selection, not a product with 0: an infinity or NaN in one
// segment reaches neither the next segment's states nor the gradients of the
// one before.
//
// A tile is 64 channels x 64 or 128 tokens, or 32 channels x 128 tokens (see
// tile_elems and geom), one CTA each: 8 row warps and a look-back warp.  A lane
// owns 4 channels (two packed fp32 pairs) of 4 or 8 consecutive rows, 8 or 16
// lanes a row.  Every row is mapped once to its part of the recurrence (phase 1),
// the maps are combined in the warp by shuffles, over the warps and the tiles
// before by the look-back warp, and the rows are finished from the carry that
// enters them (phase 2).  The forward keeps the fp32 state entering every 64th
// token ([nb, spans, C], 1/32 of one 16-bit stream); the backward runs its
// states again from there, so it reads neither h nor any gate from memory, and
// both directions stream their algorithmic bytes once: 8 and 14 B per element
// (GATED, 16 bit), 12 and 22 B (SSD).  Tiles come by TMA (streams whose rows are
// not 16-byte aligned by smaller copies into the same slots), results leave by TMA
// from the slots they were computed in.
//
// What bounds it (B200, bf16; the copy's rate is 6.55 TB/s):
//   SSD 8x2048x832     forward 40 us, 4.1 TB/s; backward 75-77 us, 3.9-4.0 TB/s
//   GATED 16x4096x1024 forward 109 us, 4.9 TB/s; backward 195 us, 4.8 TB/s (resets: 112, 204)
//   8-bit copies: SSD 8x2048x832 64 and 92 us, GATED 16x4096x1024 164 and 221 us
// Neither DRAM nor any pipe is full: a tile's life is 2 us of loads, 1 to 1.6 us
// of phase 1, 0.8 to 1.5 us until its carry is handed out (an L2 round trip to
// the tile before) and 0.3 to 1 us of phase 2, and registers and shared memory
// hold 3 or 4 such tiles on an SM.  A persistent form that loads the next tile
// during this one measured slower (gated forward 134-139 us at 3 to 4 CTAs, SSD
// forward 63 us at 2): the second stage takes residents away.  Asking L2 for the tile
// that starts 148 tiles later gave the gated forward 3 % and the others nothing, 444 later
// cost the backward 3 %: the loads' latency is not what is left.
//
// Across tiles the carry travels as in scan_kernel.cuh (single pass, decoupled
// look-back over a few tiles before and the inclusive carry of the one before
// those, composed in a fixed order, so results are bit-reproducible), but with
// its own records: 32-bit words holding the complement of a float's bits, 0 while
// unwritten.  The call clears them on its stream before the launch, so a
// workspace carries nothing from one call to the next, and graphs that captured
// calls can be replayed in any order.  Blocks start in the order of the tiles
// (chains along x, positions along y and z), so the tiles a block waits for are
// resident or finished.  Every wait is bounded; one that gives up sets a bit of the
// device's error word (need_scan_train_error) and passes NaN on.
//
// Checkpoints in 8 bits: the forward also writes its inputs as e4m3 with one
// power of two per token and 64 channels, and the backward reads those (5 + 2
// bytes per SSD element in place of 12) -- the gradient is then the formula's
// at the stored values, from the true state entering each tile.
#include <cuda_fp8.h>
#include <string.h>

#include <algorithm>
#include <type_traits>

#include "host_common.h"
#include "need_scan.h"
#include "scan_kernel.cuh"
#include "train_common.cuh"

using namespace need;

namespace {

constexpr int kGroup = 64;             // channels of a token that share an 8-bit scale
constexpr int kSpan = 64;              // tokens between kept states
constexpr int kNW = 8;                 // row warps
constexpr int kNT = (kNW + 1) * 32;    // threads: the row warps and the look-back warp
// Tokens x channels per tile.  The wide GATED scans, with little to keep per
// element, take tiles twice as long (16x4096x1024 bf16: forward 107 us against
// 130 us, the 16-bit backward, which keeps less, 191 against 209 us (f16 189, 213);
// with 8-bit copies forward 161 against 201 us, and 47 against 68 us at 1x16384x832,
// whose chains are few); the others lose more residents than they save (SSD 8x2048x832
// backward 88 against 76 us; with 8-bit copies forward 76 against 64 us, GATED backward
// 303 against 223 us at 16x4096x1024).
__host__ __device__ constexpr int tile_elems(int form, bool half, bool ck, int cb, bool bwd) {
    return form == FORM_GATED && cb == 64 && (!bwd || (half && !ck)) ? 8192 : 4096;
}
constexpr int kNear = 3, kDeep = 5;    // tile maps composed before an inclusive carry
constexpr int kHdrBytes = WS_HDR_WORDS * 4;
constexpr int kRecBytes = 12;           // per tile and channel: (A, B) and the inclusive carry

struct TrainParams {
    CUtensorMap tm[6];   // the streamed inputs, and gout (backward, last)
    CUtensorMap tmo[5];  // the streamed outputs: out, or grad[]
    uint32_t plain;      // bit k: stream k is read with plain loads, from
    const void* src[6];
    uint8_t unit[6];     // elements per such load: the largest of 4, 2, 1 that its rows allow
    int64_t ssb[6], sst[6];
    int32_t nb, T, C, ncb, nchains, nchunks;  // tiles along T
    int32_t nspans, depth, ngroups;           // kept states along T; look-back depth; 8-bit scales per token
    const float* dskip;
    float dt_min, dt_scale;
    const float* h0;       // forward: initial state; backward: unused (the states hold it)
    float* h_final;        // forward
    const uint8_t* seg;
    int64_t sgb, sgt;
    float* states;         // [nb, nspans, C] the state entering each span
    uint8_t* q;            // 8-bit values [nin][nb][T][ngroups * 64]
    uint8_t* qs;           // their scales [nin][nb][T][ngroups]
    const float* g_final;  // backward: gradient of the final state or null
    float* grad_h0;        // backward, optional
    float* dpart;          // backward SSD: [nb * nchunks, C] partial sums of the gradient of D
    uint32_t* hdr;
    unsigned long long* agg;  // [ntiles][CB] (A, B)
    uint32_t* incl;           // [ntiles][CB] the carry past the tile
    uint32_t polls, load_polls;  // before a wait for another tile's records, or for this warp's loads, gives up
};

// What the waits that gave up have set since need_scan_train_error last read it: a call's
// workspace is gone when it returns, so its own word cannot tell.
__device__ uint32_t g_train_error;
__device__ __forceinline__ void give_up(const TrainParams& p, uint32_t bit) {
    atomicOr(&p.hdr[WS_ERROR], bit);
    atomicOr(&g_train_error, bit);
}
__device__ __forceinline__ float nan32() { return __int_as_float(0x7fc00000); }

// ------------------------------------------------------------------ maps
// Affine maps c -> A c + B.  With segments in the call (`seg`), A == -0 means "drops
// c", whatever c holds.  A product of a's is never negative: one that has underflowed is
// +0, and an infinity or NaN that it multiplies stays in its segment.
__device__ __forceinline__ float2 drop2() { return splat2(-0.0f); }
__device__ __forceinline__ bool drops(float A) { return __float_as_uint(A) == 0x80000000u; }
__device__ __forceinline__ float2 apply(float2 A, float2 c, float2 B, bool seg) {
    float2 r = ffma2(A, c, B);
    if (seg) r = make_float2(drops(A.x) ? B.x : r.x, drops(A.y) ? B.y : r.y);
    return r;
}
__device__ __forceinline__ float apply(float A, float c, float B, bool seg) {
    return seg && drops(A) ? B : fmaf(A, c, B);
}
__device__ __forceinline__ float mulz(float a, float b, bool seg) {
    return seg && (drops(a) || drops(b)) ? -0.0f : a * b;
}
__device__ __forceinline__ float2 mulz(float2 a, float2 b, bool seg) {
    float2 r = fmul2(a, b);
    if (seg) r = make_float2(drops(a.x) || drops(b.x) ? -0.0f : r.x, drops(a.y) || drops(b.y) ? -0.0f : r.y);
    return r;
}

// ------------------------------------------------------------------ records
// The complement of a float's bits, two to a 64-bit word; 0 = not written yet
// (the one NaN that would read so is written as another).
__device__ __forceinline__ uint32_t rec_enc(float v) {
    const uint32_t b = ~__float_as_uint(v);
    return b == 0u ? 0x80000000u : b;
}
__device__ __forceinline__ unsigned long long rec_pair(float a, float b) {
    return (static_cast<unsigned long long>(rec_enc(b)) << 32) | rec_enc(a);
}
__device__ __forceinline__ bool rec_set(unsigned long long w) {
    return static_cast<uint32_t>(w) != 0u && static_cast<uint32_t>(w >> 32) != 0u;
}
__device__ __forceinline__ float rec_lo(unsigned long long w) { return __uint_as_float(~static_cast<uint32_t>(w)); }
__device__ __forceinline__ float rec_hi(unsigned long long w) {
    return __uint_as_float(~static_cast<uint32_t>(w >> 32));
}
__device__ __forceinline__ void st_relaxed_u64(unsigned long long* p, unsigned long long a) {
    asm volatile("st.relaxed.gpu.global.u64 [%0], %1;" ::"l"(p), "l"(a) : "memory");
}
__device__ __forceinline__ unsigned long long ld_relaxed_u64(const unsigned long long* p) {
    unsigned long long v;
    asm volatile("ld.relaxed.gpu.global.u64 %0, [%1];" : "=l"(v) : "l"(p) : "memory");
    return v;
}
__device__ __forceinline__ void st_relaxed_u32(uint32_t* p, uint32_t a) {
    asm volatile("st.relaxed.gpu.global.u32 [%0], %1;" ::"l"(p), "r"(a) : "memory");
}
__device__ __forceinline__ uint32_t ld_relaxed_u32(const uint32_t* p) {
    uint32_t v;
    asm volatile("ld.relaxed.gpu.global.u32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
    return v;
}
// A lane's NC channels of a record.
template <int NC>
struct Agg {
    unsigned long long w[NC];
    __device__ __forceinline__ void load(const unsigned long long* p) {
        if constexpr (NC == 2) {
            const ulonglong2 v = ld_relaxed_v2u64(reinterpret_cast<const ulonglong2*>(p));
            w[0] = v.x, w[1] = v.y;
        } else {
            w[0] = ld_relaxed_u64(p);
        }
    }
    __device__ __forceinline__ void store(unsigned long long* p) const {
        if constexpr (NC == 2) st_relaxed_v2u64(reinterpret_cast<ulonglong2*>(p), w[0], w[1]);
        else st_relaxed_u64(p, w[0]);
    }
    __device__ __forceinline__ bool set() const {
        bool ok = true;
#pragma unroll
        for (int k = 0; k < NC; ++k) ok &= rec_set(w[k]);
        return ok;
    }
};
template <int NC>
struct Incl {
    uint32_t w[NC];
    __device__ __forceinline__ void load(const uint32_t* p) {
        if constexpr (NC == 2) {
            const unsigned long long v = ld_relaxed_u64(reinterpret_cast<const unsigned long long*>(p));
            w[0] = static_cast<uint32_t>(v), w[1] = static_cast<uint32_t>(v >> 32);
        } else {
            w[0] = ld_relaxed_u32(p);
        }
    }
    __device__ __forceinline__ void store(uint32_t* p) const {
        if constexpr (NC == 2)
            st_relaxed_u64(reinterpret_cast<unsigned long long*>(p), (static_cast<unsigned long long>(w[1]) << 32) | w[0]);
        else st_relaxed_u32(p, w[0]);
    }
    __device__ __forceinline__ bool set() const {
        bool ok = true;
#pragma unroll
        for (int k = 0; k < NC; ++k) ok &= w[k] != 0u;
        return ok;
    }
};
template <int NC>
struct Ch {  // a lane's channels in the look-back warp
    float v[NC];
};

// ------------------------------------------------------------------ inputs
struct F4 {  // four channels
    float2 p[2];
};
// Channels 4 v .. 4 v + 3 of row r of a slot.
template <typename T, int CB>
__device__ __forceinline__ F4 row4(const unsigned char* slot, int r, int v) {
    F4 f;
    if constexpr (Ops<T>::BYTES == 4) {
        const float4 x = reinterpret_cast<const float4*>(slot)[r * (CB / 4) + v];
        f.p[0] = make_float2(x.x, x.y);
        f.p[1] = make_float2(x.z, x.w);
    } else {
        const uint2 x = reinterpret_cast<const uint2*>(slot)[r * (CB / 4) + v];
        f.p[0] = widen(*reinterpret_cast<const typename Ops<T>::P*>(&x.x));
        f.p[1] = widen(*reinterpret_cast<const typename Ops<T>::P*>(&x.y));
    }
    return f;
}
template <typename T, int CB>
__device__ __forceinline__ void put4(unsigned char* slot, int r, int v, const F4& f) {
    const typename Ops<T>::P h[2] = {Ops<T>::pack(f.p[0].x, f.p[0].y), Ops<T>::pack(f.p[1].x, f.p[1].y)};
    if constexpr (Ops<T>::BYTES == 4)
        reinterpret_cast<float4*>(slot)[r * (CB / 4) + v] = *reinterpret_cast<const float4*>(h);
    else reinterpret_cast<uint2*>(slot)[r * (CB / 4) + v] = *reinterpret_cast<const uint2*>(h);
}
// The same of an 8-bit slot, times its row's scale.
template <int CB>
__device__ __forceinline__ F4 row4_8(const unsigned char* slot, int r, int v, float scale) {
    const uint32_t q = reinterpret_cast<const uint32_t*>(slot)[r * (CB / 4) + v];
    F4 f;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const __nv_fp8x2_storage_t h = static_cast<__nv_fp8x2_storage_t>(q >> (16 * i));
        f.p[i] = fmul2(__half22float2(static_cast<__half2>(__nv_cvt_fp8x2_to_halfraw2(h, __NV_E4M3))), splat2(scale));
    }
    return f;
}

// A pair s, n = 1 - s in one number y: s where it is the smaller, else -n (s = 1: -0).
__device__ __forceinline__ float2 smaller(float2 s, float2 n) {
    return make_float2(s.x < 0.5f ? s.x : -n.x, s.y < 0.5f ? s.y : -n.y);
}
__device__ __forceinline__ float2 one_if_negative(float2 y) {  // by the sign bit: -0 too
    return make_float2(__int_as_float((__float_as_int(y.x) >> 31) & 0x3f800000),
                       __int_as_float((__float_as_int(y.y) >> 31) & 0x3f800000));
}
__device__ __forceinline__ float2 s_of(float2 y) { return fadd2(one_if_negative(y), y); }
__device__ __forceinline__ float2 n_of_s(float2 y) {
    const float2 o = one_if_negative(y);
    return make_float2((1.0f - o.x) - y.x, (1.0f - o.y) - y.y);
}

// What a sigmoid computed in phase 1 leaves in its stream's slot for phase 2, in place
// of the logit: fp32 streams the smaller of s and 1 - s, each as the exponential gives
// it, 1 - s with its sign turned; the other one follows by a subtraction that loses
// nothing (from s alone, 1 - s at a logit of 16 was off by 6 %).  A 16-bit slot cannot hold s to the precision the
// gradients are rounded to (f16 ends at 3e-8, bf16 has 8 bits): there the logit stays and
// the sigmoid is computed again (bf16 backward: SSD 8x2048x832 77 us, GATED 16x4096x1024
// 185; 75 and 182 with s kept as f16, which was wrong below 1e-5).
template <typename T>
constexpr bool kKeep = Ops<T>::BYTES == 4;
template <typename T, int CB>
__device__ __forceinline__ void keep4(unsigned char* slot, int r, int v, const F4& s, const F4& n) {
    if constexpr (kKeep<T>) {
        F4 y;
#pragma unroll
        for (int i = 0; i < 2; ++i) y.p[i] = smaller(s.p[i], n.p[i]);
        put4<float, CB>(slot, r, v, y);
    }
}
// s and s (1 - s) from a kept slot.
template <typename T, int CB>
__device__ __forceinline__ void kept4(const unsigned char* slot, int r, int v, F4& s, F4& slope) {
    static_assert(kKeep<T>, "kept as fp32");
    const F4 y = row4<float, CB>(slot, r, v);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        s.p[i] = s_of(y.p[i]);
        slope.p[i] = make_float2(fmaf(-y.p[i].x, y.p[i].x, fabsf(y.p[i].x)), fmaf(-y.p[i].y, y.p[i].y, fabsf(y.p[i].y)));
    }
}
template <typename T>
__device__ __forceinline__ F4 sig4(const F4& x) {
    F4 s;
    s.p[0] = sig_only<T>(x.p[0]);
    s.p[1] = sig_only<T>(x.p[1]);
    return s;
}
// The same of a logit whose sigmoid phase 2 uses again.
template <typename T, int CB>
__device__ __forceinline__ F4 sig4_keep(unsigned char* slot, int r, int v, const F4& x) {
    if constexpr (kKeep<T>) {
        F4 s, n;
#pragma unroll
        for (int i = 0; i < 2; ++i) sig_pair<T>(x.p[i], s.p[i], n.p[i]);
        keep4<T, CB>(slot, r, v, s, n);
        return s;
    } else {
        return sig4<T>(x);
    }
}

// DT: how the SSD form gets a = e^-r (r <= dt_max): 0 any range, 1 dt_max <= 1/4.
template <int FORM, typename T, bool CK, int DT, int CB_, bool BWD>
struct TrainCfg {
    static constexpr int NIN = FORM == FORM_GATED ? 3 : 5;
    static constexpr int IN_BYTES = (BWD && CK) ? 1 : Ops<T>::BYTES;  // per streamed input element
    static constexpr int CB = CB_, NC = CB / 32;                     // channels; of a look-back lane
    static constexpr int L = tile_elems(FORM, Ops<T>::BYTES == 2, CK, CB, BWD) / CB;
    static constexpr int R = L / kNW;                                // tokens; rows per warp
    static_assert(CB == 32 || CB == 64, "32 or 64 channels per tile");
    static_assert(BWD || !CK || CB == kGroup, "the 8-bit forward sees whole groups");
    static constexpr int LPR = CB / 4, SS = 32 / LPR, RT = R / SS;   // lanes per row, row groups, rows per thread
    static constexpr int IN_SLOT = L * CB * IN_BYTES;
    static constexpr int SLOT = L * CB * Ops<T>::BYTES;
    static constexpr int OFF_GOUT = NIN * IN_SLOT;
    // where kept sigmoids and results go: the input slots, or (8-bit inputs) slots of their own
    static constexpr bool STAGED = BWD && CK;
    static constexpr int OFF_STAGE = STAGED ? OFF_GOUT + SLOT : 0;
    static constexpr int OFF_MAP = OFF_GOUT + (BWD ? SLOT : 0) + (STAGED ? NIN * SLOT : 0);  // [NW][CB] (A, B)
    static constexpr int OFF_FWD = OFF_MAP + kNW * CB * 8;                 // BWD: [NW][CB] forward B
    static constexpr int OFF_IN = OFF_FWD + (BWD ? kNW * CB * 4 : 0);      // [NW][CB] carry entering each warp
    static constexpr int OFF_HIN = OFF_IN + kNW * CB * 4;                  // BWD: [NW][CB] state entering each warp
    static constexpr int OFF_DD = OFF_HIN + (BWD ? kNW * CB * 4 : 0);      // BWD SSD: [NW][CB] sums for D's gradient
    static constexpr int OFF_SCALE = OFF_DD + (BWD && FORM == FORM_SSD ? kNW * CB * 4 : 0);  // BWD CK: [NW][NIN][R]
    static constexpr int OFF_BAR = OFF_SCALE + (BWD && CK ? kNW * NIN * R * 4 : 0);
    static constexpr int SMEM = OFF_BAR + (kNW + 1) * 8;
    // CTAs per SM that registers are planned for (16 bit: 56 to 96 registers).  Most of
    // a tile's time is latency -- its loads 2 us, the carry 1 us -- so residents count for
    // more than a few spilled registers: SSD 8x2048x832 forward 40 us at 4, 44 at 3;
    // backward 76 at 3, 87 at 2; the GATED one of 16x4096x1024 with 8-bit copies 268 at 2,
    // 215 at 3 (before its gates were computed again: 221 now).  The SSD backward with 8-bit
    // copies: shared memory holds two tiles, of fp32 one (registers for three 102 us, for two
    // 94; fp32 for two 244, for one 238).
    static constexpr bool SSD8 = BWD && CK && FORM == FORM_SSD;
    static constexpr int MINB = Ops<T>::BYTES == 4 ? (SSD8 ? 1 : 2) : BWD ? (SSD8 ? 2 : 3) : (CK || L * CB > 4096 ? 3 : 4);
};

// ------------------------------------------------------------------ look-back
// The look-back warp's work for one tile: composes the tile's map from the
// warps' maps, publishes it, takes the carry that enters the tile, publishes
// the one that leaves it, and leaves in s_in the carry entering each warp's
// rows.  `carry` holds the initial value where pos == 0, else it is read.  REV:
// the carry meets the warps from last to first.  Returns the carry past the tile.
template <bool REV, int NC, class Wait>
__device__ __forceinline__ Ch<NC> look_back(const TrainParams& p, int64_t tile, int pos, bool last, int lane,
                                            Ch<NC>& carry, const float2* s_map, float* s_in, Wait maps_ready) {
    constexpr int CB = 32 * NC;
    const int nagg = min(pos - 1, p.depth);
    const bool seg = p.seg != nullptr;
    bool have = pos == 0, mapped = false;
    const int64_t step = int64_t(p.nchains) * CB;
    const unsigned long long* young = p.agg + (tile - p.nchains) * CB + lane * NC;
    const uint32_t* old = p.incl + (tile - int64_t(nagg + 1) * p.nchains) * CB + lane * NC;
    Ch<NC> A, B;
    // one look at the records: all of them read at once, composed if all are there
    auto look = [&](auto depth) {
        constexpr int D = decltype(depth)::value;
        Agg<NC> m[D];
        Incl<NC> c;
#pragma unroll
        for (int j = 0; j < D; ++j)
            if (j < nagg) m[j].load(young - j * step);
        c.load(old);
        bool valid = c.set();
#pragma unroll
        for (int j = 0; j < D; ++j)
            if (j < nagg) valid &= m[j].set();
        if (!__all_sync(0xffffffffu, valid)) return false;
#pragma unroll
        for (int k = 0; k < NC; ++k) {
            float accA = 1.0f, accB = 0.0f;
#pragma unroll
            for (int j = 0; j < D; ++j) {
                if (j < nagg) {
                    accB = apply(accA, rec_hi(m[j].w[k]), accB, seg);
                    accA = mulz(accA, rec_lo(m[j].w[k]), seg);
                }
            }
            carry.v[k] = apply(accA, __uint_as_float(~c.w[k]), accB, seg);
        }
        return true;
    };
    auto map_of = [&](int w, int k) { return s_map[w * CB + lane * NC + k]; };
    for (uint32_t it = 0;; ++it) {
        if (!have) have = p.depth > kNear ? look(std::integral_constant<int, kDeep>{}) : look(std::integral_constant<int, kNear>{});
        // with the carry in, nothing else is polled: suspend on the barrier
        if (!mapped && maps_ready(have)) {
#pragma unroll
            for (int k = 0; k < NC; ++k) {
                A.v[k] = 1.0f;
                B.v[k] = 0.0f;
#pragma unroll
                for (int w = 0; w < kNW; ++w) {  // in the order the carry meets the warps
                    const float2 m = map_of(REV ? kNW - 1 - w : w, k);
                    B.v[k] = apply(m.x, B.v[k], m.y, seg);
                    A.v[k] = mulz(m.x, A.v[k], seg);
                }
            }
            if (!last && pos > 0) {  // the first tile's map is never composed: its carry is known
                Agg<NC> r;
#pragma unroll
                for (int k = 0; k < NC; ++k) r.w[k] = rec_pair(A.v[k], B.v[k]);
                r.store(p.agg + tile * CB + lane * NC);
            }
            mapped = true;
        }
        if (mapped && have) break;
        if (!have && it >= p.polls) {  // go on without a predecessor's carry
            if (lane == 0) give_up(p, ERR_LOOKBACK);
#pragma unroll
            for (int k = 0; k < NC; ++k) carry.v[k] = nan32();
            have = true;
        } else if (have && it - min(it, p.polls) >= kTmaPolls) {  // without this tile's maps: NaN for all its warps
            if (lane == 0) give_up(p, ERR_TMA);
#pragma unroll
            for (int k = 0; k < NC; ++k) A.v[k] = B.v[k] = nan32();
            break;
        }
    }
    Ch<NC> past;
    Incl<NC> r;
#pragma unroll
    for (int k = 0; k < NC; ++k) {
        past.v[k] = apply(A.v[k], carry.v[k], B.v[k], seg);
        r.w[k] = rec_enc(past.v[k]);
    }
    if (!last) r.store(p.incl + tile * CB + lane * NC);
    Ch<NC> c = carry;
#pragma unroll
    for (int n = 0; n < kNW; ++n) {
        const int w = REV ? kNW - 1 - n : n;
#pragma unroll
        for (int k = 0; k < NC; ++k) {
            s_in[w * CB + lane * NC + k] = mapped ? c.v[k] : nan32();
            const float2 m = map_of(w, k);
            c.v[k] = apply(m.x, c.v[k], m.y, seg);
        }
    }
    return past;
}

// This lane's two channels of a [.., C] fp32 row (0 past C).
__device__ __forceinline__ float2 ld_pair(const float* row, int c, int C) {
    return make_float2(c < C ? row[c] : 0.0f, c + 1 < C ? row[c + 1] : 0.0f);
}
__device__ __forceinline__ float2 shfl2(float2 x, int m) {
    return make_float2(__shfl_xor_sync(0xffffffffu, x.x, m), __shfl_xor_sync(0xffffffffu, x.y, m));
}
__device__ __forceinline__ void st_pair(float* row, int c, int C, float2 v) {
    if (c < C) row[c] = v.x;
    if (c + 1 < C) row[c + 1] = v.y;
}

template <int NC>
__device__ __forceinline__ Ch<NC> ld_ch(const float* row, int c, int C) {
    Ch<NC> r;
#pragma unroll
    for (int k = 0; k < NC; ++k) r.v[k] = c + k < C ? row[c + k] : 0.0f;
    return r;
}
template <int NC>
__device__ __forceinline__ void st_ch(float* row, int c, int C, const Ch<NC>& x) {
#pragma unroll
    for (int k = 0; k < NC; ++k)
        if (c + k < C) row[c + k] = x.v[k];
}

struct Tile {
    int pos, chunk, cblk, b, t0, c0, nvalid;
    int64_t tile;
};
template <int L, int CB>
__device__ __forceinline__ Tile tile_of(const TrainParams& p, bool rev) {
    Tile t;
    // chains along x, then positions along them (y, then z): blocks start in that
    // order, so the tiles a block waits for are resident or finished
    const int chain = static_cast<int>(blockIdx.x);
    t.pos = static_cast<int>(blockIdx.y + blockIdx.z * gridDim.y);  // in the order the carry meets the tiles
    t.tile = int64_t(t.pos) * p.nchains + chain;
    t.chunk = rev ? p.nchunks - 1 - t.pos : t.pos;
    t.b = chain / p.ncb;
    t.cblk = chain - t.b * p.ncb;
    t.t0 = t.chunk * L;
    t.c0 = t.cblk * CB;
    t.nvalid = min(L, p.T - t.t0);
    return t;
}

// Bit j: row wr0 + j of the tile starts a segment (rows past T: clear).
template <int R>
__device__ __forceinline__ uint32_t reset_bits(const TrainParams& p, const Tile& tl, int wr0, int lane) {
    bool r = false;
    const int t = tl.t0 + wr0 + lane;
    if (p.seg != nullptr && lane < R && t < p.T) r = p.seg[tl.b * p.sgb + int64_t(t) * p.sgt] != 0;
    return __ballot_sync(0xffffffffu, r);
}

// A warp's rows of stream k with ordinary loads, as TMA would leave them (zeros past C
// and T), U elements each.  4 and 8 bytes are copied asynchronously, so that all streams
// are on their way together; the caller waits (SSD 8 x 2048 bf16, forward / backward us:
// C = 828, 8 bytes, 57 / 96; 830, 4 bytes, 67 / 107; 831, one element a load, 87 / 142;
// 832 by TMA 40 / 76).
template <typename T, int R, int CB, int U>
__device__ __forceinline__ void plain_units(const TrainParams& p, const Tile& tl, const T* src, int64_t st,
                                            unsigned char* slot, int rows, int lane) {
    constexpr int UR = CB / U, BYTES = U * sizeof(T);  // units in a row, bytes in a unit
    static_assert(R * UR % 32 == 0, "whole warps");
    if constexpr (BYTES >= 4) {
#pragma unroll 4
        for (int i = lane; i < R * UR; i += 32) {
            const int r = i / UR, e = U * (i - r * UR);
            const bool in = r < rows && tl.c0 + e < p.C;
            asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(smem_addr(slot + i * BYTES)),
                         "l"(in ? src + r * st + e : src), "n"(BYTES), "r"(in ? BYTES : 0)
                         : "memory");
        }
    } else {
        constexpr int G = 8;  // loads on their way at once
        static_assert(R * UR % (32 * G) == 0, "whole batches");
        for (int i0 = lane; i0 < R * UR; i0 += 32 * G) {
            T x[G];
#pragma unroll
            for (int g = 0; g < G; ++g) {
                const int i = i0 + 32 * g, r = i / UR, e = i - r * UR;
                memset(&x[g], 0, sizeof(T));
                if (r < rows && tl.c0 + e < p.C) x[g] = src[r * st + e];
            }
#pragma unroll
            for (int g = 0; g < G; ++g) reinterpret_cast<T*>(slot)[i0 + 32 * g] = x[g];
        }
    }
}
template <typename T, int R, int CB>
__device__ __forceinline__ void plain_rows(const TrainParams& p, const Tile& tl, int k, unsigned char* slot, int wr0,
                                           int rows, int lane) {
    const int64_t st = p.sst[k];
    const T* src = static_cast<const T*>(p.src[k]) + tl.b * p.ssb[k] + int64_t(tl.t0 + wr0) * st + tl.c0;
    if constexpr (sizeof(T) == 2) {
        if (p.unit[k] == 4) plain_units<T, R, CB, 4>(p, tl, src, st, slot, rows, lane);
    }
    if (p.unit[k] == 2) plain_units<T, R, CB, 2>(p, tl, src, st, slot, rows, lane);
    if (p.unit[k] == 1) plain_units<T, R, CB, 1>(p, tl, src, st, slot, rows, lane);
}

// Starts the loads of a warp's rows: n streams, of `bytes` per element (gout,
// stream n - 1 of the backward, of sizeof(T)), into slot(k).
template <typename T, int N, int NIN, int IN_BYTES, int R, int CB, class Slot>
__device__ __forceinline__ void load_rows(const TrainParams& p, const Tile& tl, int wr0, int rows, int lane,
                                          uint64_t* bar, bool stacked, Slot slot) {
    if (rows > 0) {
        if (lane == 0) {
            uint32_t tx = 0;
#pragma unroll
            for (int k = 0; k < N; ++k)
                if (!((p.plain >> k) & 1u)) tx += R * CB * (k < NIN ? IN_BYTES : Ops<T>::BYTES);
            mbar_arrive_expect_tx(bar, tx);
#pragma unroll
            for (int k = 0; k < N; ++k)
                if (!((p.plain >> k) & 1u))
                    tma_load_3d(slot(k), &p.tm[k], tl.c0, tl.t0 + wr0, stacked && k < NIN ? k * p.nb + tl.b : tl.b, bar);
        }
        if (p.plain != 0) {
            for (int k = 0; k < N; ++k)
                if ((p.plain >> k) & 1u) plain_rows<T, R, CB>(p, tl, k, slot(k), wr0, rows, lane);
            asm volatile("cp.async.wait_all;" ::: "memory");
            __syncwarp();
        }
    }
}

// Waits for them.  Rows whose wait runs out become NaN in every stream (all bits set, in
// e4m3 too), and with them whatever depends on them -- once the copies have landed, which
// a second wait gives them time for.
template <typename T, int N, int NIN, int IN_BYTES, int R, int CB, class Slot>
__device__ __forceinline__ void await_rows(const TrainParams& p, int rows, int lane, uint64_t* bar, Slot slot) {
    const bool late = rows > 0 && !mbar_wait_bounded(bar, 0, p.load_polls);
    if (__any_sync(0xffffffffu, late)) {
        if (lane == 0) give_up(p, ERR_TMA);
        mbar_wait_bounded(bar, 0, kTmaPolls);
        for (int k = 0; k < N; ++k)
            for (int i = lane; i < R * CB * (k < NIN ? IN_BYTES : int(sizeof(T))) / 4; i += 32)
                reinterpret_cast<uint32_t*>(slot(k))[i] = ~0u;
        __syncwarp();
    }
}

// a and 1 - a of the decay stream's four channels, and of the SSD form's step s and (PAIR) 1 - s.
template <int FORM, typename T, int DT, bool PAIR>
__device__ __forceinline__ void decay4(const TrainParams& p, const F4& x, F4& a, F4& na, F4& s, F4& ns) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        if constexpr (FORM == FORM_GATED) {
            sig_pair<T>(x.p[i], a.p[i], na.p[i]);
        } else {
            if constexpr (PAIR) sig_pair<T>(x.p[i], s.p[i], ns.p[i]);
            else s.p[i] = sig_only<T>(x.p[i]);
            const float2 r = ffma2(s.p[i], splat2(p.dt_scale), splat2(p.dt_min));
            if constexpr (DT == 1) exp_neg_small(r, a.p[i], na.p[i]);
            else exp_neg<T>(r, a.p[i], na.p[i]);
        }
    }
}

// The 8-bit copies of a warp's rows: a lane takes 16 bytes, 64 channels lie in
// 64 / N neighbouring lanes.
template <typename T, int NIN, int R>
__device__ __forceinline__ void write_e4m3(const TrainParams& p, const Tile& tl, const unsigned char* base, int slot_bytes,
                                           int wr0, int rows, int lane) {
    constexpr int N = 16 / Ops<T>::BYTES, LPR = kGroup / N, RP = 32 / LPR;  // elements, lanes per row, rows at once
    const int v = lane % LPR;
    // this lane's first row of stream 0, and the way to the next rows and streams
    const int64_t first = int64_t(tl.b) * p.T + tl.t0 + wr0 + lane / LPR, stream = int64_t(p.nb) * p.T;
    const int pitch = p.ngroups * kGroup;
    uint8_t* dst0 = p.q + first * pitch + tl.c0 + v * N;
    uint8_t* sc0 = p.qs + first * p.ngroups + tl.cblk;
#pragma unroll
    for (int k = 0; k < NIN; ++k, dst0 += stream * pitch, sc0 += stream * p.ngroups) {
        const unsigned char* slot = base + k * slot_bytes;
        uint8_t *dst = dst0, *scp = sc0;
#pragma unroll
        for (int r0 = 0; r0 < R; r0 += RP, dst += RP * pitch, scp += RP * p.ngroups) {
            const int r = r0 + lane / LPR;
            const uint4 raw = reinterpret_cast<const uint4*>(slot)[r * LPR + v];
            const typename Ops<T>::P* h = reinterpret_cast<const typename Ops<T>::P*>(&raw);
            float2 f[N / 2];
            uint32_t top;
#pragma unroll
            for (int e = 0; e < N / 2; ++e) f[e] = widen(h[e]);
            if constexpr (Ops<T>::BYTES == 2) {
                // magnitudes of 16-bit floats order as their bits do
                const uint32_t w[4] = {raw.x & 0x7fff7fffu, raw.y & 0x7fff7fffu, raw.z & 0x7fff7fffu, raw.w & 0x7fff7fffu};
                uint32_t m = __vmaxu2(__vmaxu2(w[0], w[1]), __vmaxu2(w[2], w[3]));
#pragma unroll
                for (int d = LPR / 2; d >= 1; d >>= 1) m = __vmaxu2(m, __shfl_xor_sync(0xffffffffu, m, d));
                const uint16_t b = static_cast<uint16_t>(max(m & 0xffffu, m >> 16));
                if constexpr (std::is_same<T, __half>::value) top = __float_as_uint(__half2float(__ushort_as_half(b)));
                else top = static_cast<uint32_t>(b) << 16;
            } else {
                top = 0;
#pragma unroll
                for (int e = 0; e < N / 2; ++e)
                    top = max(top, max(__float_as_uint(f[e].x) & 0x7fffffffu, __float_as_uint(f[e].y) & 0x7fffffffu));
#pragma unroll
                for (int d = LPR / 2; d >= 1; d >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, d));
            }
            const uint32_t sc = e4m3_scale_byte(top);
            const float inv = e4m3_inverse(sc);
            uint32_t q[N / 4];
#pragma unroll
            for (int e = 0; e < N / 4; ++e)
                q[e] = e4m3_round(fmul2(f[2 * e], splat2(inv))) | uint32_t(e4m3_round(fmul2(f[2 * e + 1], splat2(inv)))) << 16;
            if (r < rows) {
                if constexpr (N == 8) *reinterpret_cast<uint2*>(dst) = make_uint2(q[0], q[1]);
                else *reinterpret_cast<uint32_t*>(dst) = q[0];
                if (v == 0) *scp = static_cast<uint8_t>(sc);
            }
        }
    }
}

// ------------------------------------------------------------------ in-warp scan
template <class Shfl>
__device__ __forceinline__ F4 shfl4(const F4& x, Shfl f) {
    F4 r;
#pragma unroll
    for (int i = 0; i < 2; ++i) r.p[i] = make_float2(f(x.p[i].x), f(x.p[i].y));
    return r;
}
// The SS row groups of a warp hold consecutive rows.  In: each thread's map of its
// rows.  Out: (A, B) of its and the groups' before it, (EA, EB) of those before
// it alone.  The last group's (A, B) is the warp's.
template <int LPR, int SS>
__device__ __forceinline__ void warp_prefix(F4& A, F4& B, F4& EA, F4& EB, int q, bool seg) {
    F4 oA, oB;
#pragma unroll
    for (int d = 1; d < SS; d *= 2) {
        oA = shfl4(A, [&](float x) { return __shfl_up_sync(0xffffffffu, x, d * LPR); });
        oB = shfl4(B, [&](float x) { return __shfl_up_sync(0xffffffffu, x, d * LPR); });
        if (q >= d) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                B.p[i] = apply(A.p[i], oB.p[i], B.p[i], seg);
                A.p[i] = mulz(A.p[i], oA.p[i], seg);
            }
        }
    }
    if constexpr (SS == 2) {
        EA = oA, EB = oB;
    } else {
        EA = shfl4(A, [&](float x) { return __shfl_up_sync(0xffffffffu, x, LPR); });
        EB = shfl4(B, [&](float x) { return __shfl_up_sync(0xffffffffu, x, LPR); });
    }
    if (q == 0) {
#pragma unroll
        for (int i = 0; i < 2; ++i) EA.p[i] = splat2(1.0f), EB.p[i] = splat2(0.0f);
    }
}
// The same from the last group to the first: the carry enters the last.
template <int LPR, int SS>
__device__ __forceinline__ void warp_suffix(F4& A, F4& M, F4& EA, F4& EM, int q, bool seg) {
    F4 oA, oM;
#pragma unroll
    for (int d = 1; d < SS; d *= 2) {
        oA = shfl4(A, [&](float x) { return __shfl_down_sync(0xffffffffu, x, d * LPR); });
        oM = shfl4(M, [&](float x) { return __shfl_down_sync(0xffffffffu, x, d * LPR); });
        if (q + d < SS) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                M.p[i] = apply(A.p[i], oM.p[i], M.p[i], seg);
                A.p[i] = mulz(A.p[i], oA.p[i], seg);
            }
        }
    }
    if constexpr (SS == 2) {
        EA = oA, EM = oM;
    } else {
        EA = shfl4(A, [&](float x) { return __shfl_down_sync(0xffffffffu, x, LPR); });
        EM = shfl4(M, [&](float x) { return __shfl_down_sync(0xffffffffu, x, LPR); });
    }
    if (q == SS - 1) {
#pragma unroll
        for (int i = 0; i < 2; ++i) EA.p[i] = splat2(1.0f), EM.p[i] = splat2(0.0f);
    }
}
__device__ __forceinline__ void put_maps(float2* dst, const F4& A, const F4& B) {
    float4* d = reinterpret_cast<float4*>(dst);
#pragma unroll
    for (int i = 0; i < 2; ++i) d[i] = make_float4(A.p[i].x, B.p[i].x, A.p[i].y, B.p[i].y);
}
__device__ __forceinline__ float4 as_float4(const F4& x) { return make_float4(x.p[0].x, x.p[0].y, x.p[1].x, x.p[1].y); }

// The forward's product of a up to a row, kept from phase 1 to phase 2 in fp32 (held in
// f16 it loses its last bits, and all of them below 6e-8).  In place of the logits of
// streams 0 and 1, which phase 2 does not read: their two 16-bit slots hold the upper
// and the lower halves, so that it costs no registers.
template <typename T, int CB>
__device__ __forceinline__ void put_prod(unsigned char* slot0, unsigned char* slot1, int r, int v, const F4& x) {
    if constexpr (Ops<T>::BYTES == 4) {
        put4<float, CB>(slot0, r, v, x);
    } else {
        const uint32_t w[4] = {__float_as_uint(x.p[0].x), __float_as_uint(x.p[0].y), __float_as_uint(x.p[1].x),
                               __float_as_uint(x.p[1].y)};
        reinterpret_cast<uint2*>(slot0)[r * (CB / 4) + v] =
            make_uint2(__byte_perm(w[0], w[1], 0x7632), __byte_perm(w[2], w[3], 0x7632));
        reinterpret_cast<uint2*>(slot1)[r * (CB / 4) + v] =
            make_uint2(__byte_perm(w[0], w[1], 0x5410), __byte_perm(w[2], w[3], 0x5410));
    }
}
template <typename T, int CB>
__device__ __forceinline__ F4 get_prod(const unsigned char* slot0, const unsigned char* slot1, int r, int v) {
    if constexpr (Ops<T>::BYTES == 4) {
        return row4<float, CB>(slot0, r, v);
    } else {
        const uint2 hi = reinterpret_cast<const uint2*>(slot0)[r * (CB / 4) + v];
        const uint2 lo = reinterpret_cast<const uint2*>(slot1)[r * (CB / 4) + v];
        F4 x;
        x.p[0] = make_float2(__uint_as_float(__byte_perm(lo.x, hi.x, 0x5410)), __uint_as_float(__byte_perm(lo.x, hi.x, 0x7632)));
        x.p[1] = make_float2(__uint_as_float(__byte_perm(lo.y, hi.y, 0x5410)), __uint_as_float(__byte_perm(lo.y, hi.y, 0x7632)));
        return x;
    }
}

// ------------------------------------------------------------------ forward
template <int FORM, typename T, bool CK, int DT, int CBW>
__global__ void __launch_bounds__(kNT, (TrainCfg<FORM, T, CK, DT, CBW, false>::MINB))
    train_fwd_kernel(const __grid_constant__ TrainParams p) {
    using K = TrainCfg<FORM, T, CK, DT, CBW, false>;
    extern __shared__ __align__(128) unsigned char base[];
    float2* s_map = reinterpret_cast<float2*>(base + K::OFF_MAP);
    float* s_in = reinterpret_cast<float*>(base + K::OFF_IN);
    uint64_t* s_bar = reinterpret_cast<uint64_t*>(base + K::OFF_BAR);
    uint64_t* s_maps = s_bar + kNW;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const bool seg = p.seg != nullptr;
    const Tile tl = tile_of<K::L, K::CB>(p, false);
    if (tl.pos >= p.nchunks) return;
    if (threadIdx.x == 0) {
        for (int w = 0; w < kNW; ++w) mbar_init(&s_bar[w], 1);
        mbar_init(s_maps, kNW * 32);
        fence_barrier_init();
    }
    __syncthreads();

    if (warp == kNW) {
        const int c = tl.c0 + K::NC * lane;
        const bool last = tl.chunk + 1 == p.nchunks;
        Ch<K::NC> carry{};
        if (tl.pos == 0 && p.h0 != nullptr) carry = ld_ch<K::NC>(p.h0 + int64_t(tl.b) * p.C, c, p.C);
        const Ch<K::NC> past =
            look_back<false, K::NC>(p, tl.tile, tl.pos, last, lane, carry, s_map, s_in, [&](bool block) {
                return __all_sync(0xffffffffu, block ? mbar_try_wait(s_maps, 0) : mbar_test_wait(s_maps, 0));
            });
        __syncwarp();
        named_arrive(1, kNT);
        float* st = p.states + (int64_t(tl.b) * p.nspans + tl.t0 / kSpan) * p.C;
        st_ch(st, c, p.C, carry);
#pragma unroll
        for (int m = 1; m < K::L / kSpan; ++m)  // the spans that start inside the tile
            if (tl.nvalid > m * kSpan)
                st_ch(st + int64_t(m) * p.C, c, p.C,
                      *reinterpret_cast<const Ch<K::NC>*>(s_in + m * kSpan / K::R * K::CB + K::NC * lane));
        if (last && p.h_final != nullptr) st_ch(p.h_final + int64_t(tl.b) * p.C, c, p.C, past);
        return;
    }

    constexpr int RT = K::RT, LPR = K::LPR, SS = K::SS, CB = K::CB;
    const int wr0 = warp * K::R;
    const int rows = max(0, min(K::R, tl.nvalid - wr0));
    unsigned char* slots = base + wr0 * K::CB * K::IN_BYTES;  // this warp's rows of stream 0
    auto slot = [&](int k) { return slots + k * K::IN_SLOT; };
    load_rows<T, K::NIN, K::NIN, K::IN_BYTES, K::R, K::CB>(p, tl, wr0, rows, lane, &s_bar[warp], false, slot);
    const uint32_t wresets = reset_bits<K::R>(p, tl, wr0, lane);
    const int q = lane / LPR, v = lane % LPR;  // row group and four channels
    const int c = tl.c0 + 4 * v;
    const uint32_t resets = (wresets >> (RT * q)) & ((1u << RT) - 1u);
    F4 D;
    if constexpr (FORM == FORM_SSD) {
        D.p[0] = ld_pair(p.dskip, c, p.C);
        D.p[1] = ld_pair(p.dskip, c + 2, p.C);
    }
    await_rows<T, K::NIN, K::NIN, K::IN_BYTES, K::R, K::CB>(p, rows, lane, &s_bar[warp], slot);

    // The copies before phase 1, which writes into the slots they are made from: they
    // delay the tile's map, but kept in registers the products spill (GATED 16x4096x1024
    // bf16 223 us against 161, on short tiles 194; SSD 8x2048x832 68 against 64).
    if constexpr (CK) {
        if (rows > 0) write_e4m3<T, K::NIN, K::R>(p, tl, slots, K::IN_SLOT, wr0, rows, lane);
        __syncwarp();
    }

    // phase 1: each row's state from a zero entering state (H) and the product
    // of a up to it (put_prod); the last are the thread's map.  Rows past T pass the
    // state on; a reset drops it.
    F4 H[RT], A, B;
#pragma unroll
    for (int i = 0; i < 2; ++i) A.p[i] = splat2(1.0f), B.p[i] = splat2(0.0f);
    auto phase1 = [&](auto whole) {
#pragma unroll
        for (int j = 0; j < RT; ++j) {
            const int r = q * RT + j;
            F4 a, na, s, ns;
            decay4<FORM, T, DT, false>(p, row4<T, CB>(slot(0), r, v), a, na, s, ns);
            const F4 g = sig4<T>(row4<T, CB>(slot(1), r, v)), x = row4<T, CB>(slot(2), r, v);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const float2 b = fmul2(na.p[i], fmul2(g.p[i], x.p[i]));
                if constexpr (decltype(whole)::value) {
                    B.p[i] = j == 0 ? b : ffma2(a.p[i], B.p[i], b);
                    A.p[i] = j == 0 ? a.p[i] : fmul2(a.p[i], A.p[i]);
                } else if (r < rows) {
                    const bool cut = ((resets >> j) & 1u) != 0u;
                    B.p[i] = cut ? b : ffma2(a.p[i], B.p[i], b);
                    A.p[i] = (resets & ((2u << j) - 1u)) != 0u ? drop2() : fmul2(a.p[i], A.p[i]);
                }
                H[j].p[i] = B.p[i];
            }
            put_prod<T, CB>(slot(0), slot(1), r, v, A);
        }
    };
    const bool whole = rows == K::R && wresets == 0u;
    if (whole) phase1(std::true_type{});
    else if (rows > 0) phase1(std::false_type{});
    F4 EA, EB;  // the map of the warp's rows before this thread's
    warp_prefix<LPR, SS>(A, B, EA, EB, q, seg);
    if (q == SS - 1) put_maps(s_map + warp * CB + 4 * v, A, B);
    mbar_arrive(s_maps);
    named_sync(1, kNT);
    if (rows == 0) return;

    // phase 2: the states from the entering one, and the outputs
    const float4 in4 = reinterpret_cast<const float4*>(s_in)[warp * LPR + v];
    F4 h0;
    h0.p[0] = apply(EA.p[0], make_float2(in4.x, in4.y), EB.p[0], seg);
    h0.p[1] = apply(EA.p[1], make_float2(in4.z, in4.w), EB.p[1], seg);
    constexpr int OUT = K::NIN - 1;  // results replace the last stream
    auto phase2 = [&](auto whole) {
#pragma unroll
        for (int j = 0; j < RT; ++j) {
            const int r = q * RT + j;
            const F4 P = get_prod<T, CB>(slot(0), slot(1), r, v);
            F4 o, sc, so, u;
            if constexpr (FORM == FORM_SSD) {
                sc = sig4<T>(row4<T, CB>(slot(3), r, v));
                so = sig4<T>(row4<T, CB>(slot(4), r, v));
                u = row4<T, CB>(slot(2), r, v);
            }
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                o.p[i] = ffma2(P.p[i], h0.p[i], H[j].p[i]);
                if constexpr (!decltype(whole)::value)
                    if ((resets & ((2u << j) - 1u)) != 0u) o.p[i] = H[j].p[i];
                if constexpr (FORM == FORM_SSD)
                    o.p[i] = fmul2(ffma2(sc.p[i], o.p[i], fmul2(D.p[i], u.p[i])), so.p[i]);
            }
            put4<T, CB>(slot(OUT), r, v, o);
        }
    };
    if (whole) phase2(std::true_type{});
    else phase2(std::false_type{});
    fence_proxy_async_shared();
    __syncwarp();
    if (lane == 0) {
        tma_store_3d(&p.tmo[0], slot(OUT), tl.c0, tl.t0 + wr0, tl.b);
        tma_store_commit();
        tma_store_drain();
    }
}

// ------------------------------------------------------------------ backward
template <int FORM, typename T, bool CK, int DT, int CBW>
__global__ void __launch_bounds__(kNT, (TrainCfg<FORM, T, CK, DT, CBW, true>::MINB))
    train_bwd_kernel(const __grid_constant__ TrainParams p) {
    using K = TrainCfg<FORM, T, CK, DT, CBW, true>;
    using O = Ops<T>;
    // The long tiles of 16-bit GATED: a is computed again for the states and in phase 2, and
    // neither it nor 1 - a is kept (16x4096x1024 191 us; kept in registers 209 on short tiles
    // and on long ones, in the logits' slots and registers 220 against 195).  The
    // SSD form loses by it (75.5 against 72.8 us), and so do the 8-bit copies (226, 223).
    constexpr bool LEAN = FORM == FORM_GATED && Ops<T>::BYTES == 2 && !CK;
    extern __shared__ __align__(128) unsigned char base[];
    float2* s_map = reinterpret_cast<float2*>(base + K::OFF_MAP);
    float* s_fwd = reinterpret_cast<float*>(base + K::OFF_FWD);
    float* s_in = reinterpret_cast<float*>(base + K::OFF_IN);
    float* s_hin = reinterpret_cast<float*>(base + K::OFF_HIN);
    float* s_dd = reinterpret_cast<float*>(base + K::OFF_DD);
    float* s_scale = reinterpret_cast<float*>(base + K::OFF_SCALE);
    uint64_t* s_bar = reinterpret_cast<uint64_t*>(base + K::OFF_BAR);
    uint64_t* s_maps = s_bar + kNW;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const bool seg = p.seg != nullptr;
    const Tile tl = tile_of<K::L, K::CB>(p, true);
    if (tl.pos >= p.nchunks) return;
    if (threadIdx.x == 0) {
        for (int w = 0; w < kNW; ++w) mbar_init(&s_bar[w], 1);
        mbar_init(s_maps, kNW * 32);
        fence_barrier_init();
    }
    __syncthreads();

    if (warp == kNW) {
        const int c = tl.c0 + K::NC * lane;
        const bool last = tl.chunk == 0;
        const float* st = p.states + (int64_t(tl.b) * p.nspans + tl.t0 / kSpan) * p.C;
        Ch<K::NC> kept[K::L / kSpan], carry{};
#pragma unroll
        for (int m = 0; m < K::L / kSpan; ++m)
            kept[m] = tl.nvalid > m * kSpan ? ld_ch<K::NC>(st + int64_t(m) * p.C, c, p.C) : Ch<K::NC>{};
        if (tl.pos == 0 && p.g_final != nullptr) carry = ld_ch<K::NC>(p.g_final + int64_t(tl.b) * p.C, c, p.C);
        bool handed = false;
        const Ch<K::NC> past =
            look_back<true, K::NC>(p, tl.tile, tl.pos, last, lane, carry, s_map, s_in, [&](bool block) {
                const bool ready =
                    __all_sync(0xffffffffu, block ? mbar_try_wait(s_maps, 0) : mbar_test_wait(s_maps, 0));
                if (ready) {  // the states entering the warps first: they wait for no other tile
                    handed = true;
                    Ch<K::NC> h = kept[0];
#pragma unroll
                    for (int w = 0; w < kNW; ++w) {
                        if (w * K::R % kSpan == 0) h = kept[w * K::R / kSpan];
#pragma unroll
                        for (int k = 0; k < K::NC; ++k) {
                            const int e = w * K::CB + K::NC * lane + k;
                            s_hin[e] = h.v[k];
                            h.v[k] = apply(s_map[e].x, h.v[k], s_fwd[e], seg);
                        }
                    }
                    __syncwarp();
                    named_arrive(1, kNT);
                }
                return ready;
            });
        if (!handed) {  // gave up: the row warps are let go, with NaN
#pragma unroll
            for (int w = 0; w < kNW; ++w)
#pragma unroll
                for (int k = 0; k < K::NC; ++k) s_hin[w * K::CB + K::NC * lane + k] = nan32();
            __syncwarp();
            named_arrive(1, kNT);
        }
        __syncwarp();
        named_arrive(2, kNT);
        if (last && p.grad_h0 != nullptr) st_ch(p.grad_h0 + int64_t(tl.b) * p.C, c, p.C, past);
        return;
    }

    constexpr int RT = K::RT, LPR = K::LPR, SS = K::SS, CB = K::CB;
    const int wr0 = warp * K::R;
    const int rows = max(0, min(K::R, tl.nvalid - wr0));
    auto slot = [&](int k) {
        return k < K::NIN ? base + k * K::IN_SLOT + wr0 * K::CB * K::IN_BYTES : base + K::OFF_GOUT + wr0 * K::CB * O::BYTES;
    };
    auto stage = [&](int k) {  // kept sigmoids, then gradients
        return K::STAGED ? base + K::OFF_STAGE + k * K::SLOT + wr0 * K::CB * O::BYTES : slot(k);
    };
    load_rows<T, K::NIN + 1, K::NIN, K::IN_BYTES, K::R, K::CB>(p, tl, wr0, rows, lane, &s_bar[warp], CK, slot);
    const uint32_t wresets = reset_bits<K::R>(p, tl, wr0, lane);
    if constexpr (CK) {
        for (int i = lane; i < K::NIN * K::R; i += 32) {
            const int k = i / K::R, j = i - k * K::R;
            float f = 0.0f;
            if (j < rows)
                f = e4m3_scale(p.qs[((int64_t(k) * p.nb + tl.b) * p.T + tl.t0 + wr0 + j) * p.ngroups + tl.c0 / kGroup]);
            s_scale[warp * K::NIN * K::R + i] = f;
        }
        __syncwarp();
    }
    const int q = lane / LPR, v = lane % LPR;
    const int c = tl.c0 + 4 * v;
    const uint32_t resets = (wresets >> (RT * q)) & ((1u << RT) - 1u);
    F4 D;
    if constexpr (FORM == FORM_SSD) {
        D.p[0] = ld_pair(p.dskip, c, p.C);
        D.p[1] = ld_pair(p.dskip, c + 2, p.C);
    }
    await_rows<T, K::NIN + 1, K::NIN, K::IN_BYTES, K::R, K::CB>(p, rows, lane, &s_bar[warp], slot);
    auto input = [&](int k, int r) {
        if constexpr (CK) return row4_8<CB>(slot(k), r, v, s_scale[(warp * K::NIN + k) * K::R + r]);
        else return row4<T, CB>(slot(k), r, v);
    };
    auto gout = [&](int r) { return row4<T, CB>(slot(K::NIN), r, v); };
    // sigmoid of logit stream k again (or as kept), and its slope
    auto gate = [&](int k, int r, F4& s, F4& slope) {
        if constexpr (kKeep<T>) {
            kept4<T, CB>(stage(k), r, v, s, slope);
        } else {
            const F4 x = input(k, r);
#pragma unroll
            for (int i = 0; i < 2; ++i) sig_slope<T>(x.p[i], s.p[i], slope.p[i]);
        }
    };

    // phase 1: the thread's maps.  Forward: h_out = A h_in + B.  Backward, over
    // the same a: mu_first = A mu_in + M, M = sum over rows of (product of a up
    // to the row) e.  The smaller of a and 1 - a stays in registers (the other one
    // follows without a loss), b too, where the states then take its place.
    F4 ka[LEAN ? 1 : RT], h[RT], A, B, M, dD;
#pragma unroll
    for (int i = 0; i < 2; ++i) A.p[i] = splat2(1.0f), B.p[i] = M.p[i] = dD.p[i] = splat2(0.0f);
    auto one_minus = [](float2 x) { return fadd2(splat2(1.0f), make_float2(-x.x, -x.y)); };
    constexpr bool NEAR1 = FORM == FORM_SSD && DT == 1;  // a >= e^-1/4: it follows from 1 - a
    auto keep_a = [&](float2 a, float2 n) { return NEAR1 ? n : smaller(a, n); };
    auto a_of = [&](float2 y) { return NEAR1 ? one_minus(y) : s_of(y); };
    auto n_of = [&](float2 y) { return NEAR1 ? y : n_of_s(y); };
    auto phase1 = [&](auto whole) {
#pragma unroll
        for (int j = 0; j < RT; ++j) {
            const int r = q * RT + j;
            F4 a, na, sd, nd;
            decay4<FORM, T, DT, kKeep<T>>(p, input(0, r), a, na, sd, nd);
            const F4 g = sig4_keep<T, CB>(stage(1), r, v, input(1, r)), x = input(2, r);
            F4 e = gout(r);
            if constexpr (FORM == FORM_SSD) {
                const F4 sc = sig4_keep<T, CB>(stage(3), r, v, input(3, r));
                const F4 so = sig4_keep<T, CB>(stage(4), r, v, input(4, r));
                keep4<T, CB>(stage(0), r, v, sd, nd);
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const float2 gs = fmul2(e.p[i], so.p[i]);
                    dD.p[i] = ffma2(gs, x.p[i], dD.p[i]);  // fp32 results come from the sigmoids as computed
                    e.p[i] = fmul2(gs, sc.p[i]);
                }
            }
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const float2 b = fmul2(na.p[i], fmul2(g.p[i], x.p[i]));
                if constexpr (!LEAN) ka[j].p[i] = keep_a(a.p[i], na.p[i]);
                h[j].p[i] = b;
                if constexpr (decltype(whole)::value) {
                    B.p[i] = j == 0 ? b : ffma2(a.p[i], B.p[i], b);
                    A.p[i] = j == 0 ? a.p[i] : fmul2(a.p[i], A.p[i]);
                    M.p[i] = j == 0 ? fmul2(A.p[i], e.p[i]) : ffma2(A.p[i], e.p[i], M.p[i]);
                } else if (r < rows) {
                    B.p[i] = ((resets >> j) & 1u) != 0u ? b : ffma2(a.p[i], B.p[i], b);
                    if ((resets & ((2u << j) - 1u)) != 0u) {
                        A.p[i] = drop2();
                    } else {
                        A.p[i] = fmul2(a.p[i], A.p[i]);
                        M.p[i] = ffma2(A.p[i], e.p[i], M.p[i]);
                    }
                }
            }
        }
    };
    const bool whole = rows == K::R && wresets == 0u;
    if (whole) phase1(std::true_type{});
    else if (rows > 0) phase1(std::false_type{});
    if constexpr (FORM == FORM_SSD) {
#pragma unroll
        for (int d = LPR; d < 32; d *= 2)
#pragma unroll
            for (int i = 0; i < 2; ++i) dD.p[i] = fadd2(dD.p[i], shfl2(dD.p[i], d));
        if (q == 0) reinterpret_cast<float4*>(s_dd)[warp * LPR + v] = as_float4(dD);
    }
    // the maps of the warp's rows before this thread's (pA, pB: the state enters
    // through them) and after them (fA, fM: mu does)
    F4 pA, pB, fA, fM, SA = A;
    warp_suffix<LPR, SS>(SA, M, fA, fM, q, seg);
    warp_prefix<LPR, SS>(A, B, pA, pB, q, seg);
    if (q == 0) put_maps(s_map + warp * CB + 4 * v, SA, M);
    if (q == SS - 1) reinterpret_cast<float4*>(s_fwd)[warp * LPR + v] = as_float4(B);
    mbar_arrive(s_maps);
    named_sync(1, kNT);

    // the states of the thread's rows, from the one entering them
    F4 hin;
    {
        const float4 in4 = reinterpret_cast<const float4*>(s_hin)[warp * LPR + v];
        hin.p[0] = make_float2(in4.x, in4.y);
        hin.p[1] = make_float2(in4.z, in4.w);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            hin.p[i] = apply(pA.p[i], hin.p[i], pB.p[i], seg);
            float2 hp = hin.p[i];
            if (rows > 0) {
#pragma unroll
                for (int j = 0; j < RT; ++j) {
                    float2 a;
                    if constexpr (LEAN) a = sig_only<T>(input(0, q * RT + j).p[i]);
                    else a = a_of(ka[j].p[i]);
                    hp = h[j].p[i] = ((resets >> j) & 1u) != 0u ? h[j].p[i] : ffma2(a, hp, h[j].p[i]);
                }
            }
        }
    }
    named_sync(2, kNT);

    // phase 2: the rows from last to first
    F4 mu;
    {
        const float4 in4 = reinterpret_cast<const float4*>(s_in)[warp * LPR + v];
        mu.p[0] = make_float2(in4.x, in4.y);
        mu.p[1] = make_float2(in4.z, in4.w);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            mu.p[i] = apply(fA.p[i], mu.p[i], fM.p[i], seg);
        }
    }
    auto phase2 = [&](auto whole) {
#pragma unroll
        for (int j = RT - 1; j >= 0; --j) {
            const int r = q * RT + j;
            if (!decltype(whole)::value && r >= rows) continue;
            const bool reset = !decltype(whole)::value && ((resets >> j) & 1u) != 0u;
            F4 sg, lg, val = input(2, r), e = gout(r), gs, d[5];
            gate(1, r, sg, lg);
            if constexpr (FORM == FORM_SSD) {
                F4 sc, lc, so, lo;
                gate(3, r, sc, lc);
                gate(4, r, so, lo);
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const float2 go = e.p[i];
                    gs.p[i] = fmul2(go, so.p[i]);
                    e.p[i] = fmul2(gs.p[i], sc.p[i]);
                    d[3].p[i] = fmul2(fmul2(gs.p[i], h[j].p[i]), lc.p[i]);
                    d[4].p[i] = fmul2(fmul2(go, ffma2(sc.p[i], h[j].p[i], fmul2(D.p[i], val.p[i]))), lo.p[i]);
                }
                put4<T, CB>(stage(3), r, v, d[3]);
                put4<T, CB>(stage(4), r, v, d[4]);
            }
            F4 sd, ld, nd, aj, nj;
            if constexpr (FORM == FORM_SSD) gate(0, r, sd, ld);
            if constexpr (LEAN) decay4<FORM, T, DT, false>(p, input(0, r), aj, nj, sd, nd);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const F4& k = ka[LEAN ? 0 : j];
                const float2 a = LEAN ? aj.p[i] : a_of(k.p[i]), n = LEAN ? nj.p[i] : n_of(k.p[i]);
                const float2 prev = reset ? splat2(0.0f) : (j > 0 ? h[j > 0 ? j - 1 : 0].p[i] : hin.p[i]);
                const float2 lam = fadd2(e.p[i], mu.p[i]);
                mu.p[i] = reset ? splat2(0.0f) : fmul2(a, lam);
                const float2 w = fmul2(sg.p[i], val.p[i]);
                const float2 da = fmul2(fmul2(lam, a), fadd2(prev, make_float2(-w.x, -w.y)));
                const float2 dw = fmul2(lam, n);
                d[1].p[i] = fmul2(fmul2(dw, val.p[i]), lg.p[i]);
                if constexpr (FORM == FORM_GATED) {
                    d[0].p[i] = fmul2(da, n);
                    d[2].p[i] = fmul2(dw, sg.p[i]);
                } else {
                    d[0].p[i] = fmul2(da, fmul2(ld.p[i], splat2(-p.dt_scale)));
                    d[2].p[i] = ffma2(dw, sg.p[i], fmul2(D.p[i], gs.p[i]));
                }
            }
            put4<T, CB>(stage(0), r, v, d[0]);
            put4<T, CB>(stage(1), r, v, d[1]);
            put4<T, CB>(stage(2), r, v, d[2]);
        }
    };
    if (whole) phase2(std::true_type{});
    else if (rows > 0) phase2(std::false_type{});
    fence_proxy_async_shared();
    __syncwarp();
    if (lane == 0 && rows > 0) {
#pragma unroll
        for (int k = 0; k < K::NIN; ++k) tma_store_3d(&p.tmo[k], stage(k), tl.c0, tl.t0 + wr0, tl.b);
        tma_store_commit();
    }
    if constexpr (FORM == FORM_SSD) {
        // the tile's sum for the gradient of D, over its warps in a fixed order (their
        // parts are there since the barriers above)
        if (warp == kNW - 1) {
            const int e = K::NC * lane;
            Ch<K::NC> sum{};
#pragma unroll
            for (int k = 0; k < K::NC; ++k)
#pragma unroll
                for (int w = 0; w < kNW; ++w) sum.v[k] += s_dd[w * CB + e + k];
            st_ch(p.dpart + (int64_t(tl.b) * p.nchunks + tl.chunk) * p.C, tl.c0 + e, p.C, sum);
        }
    }
    if (lane == 0 && rows > 0) tma_store_drain();
}

// ------------------------------------------------------------------ launch
constexpr unsigned kMaxGridY = 65535;
std::atomic<bool> g_load_give_up{false};  // need_test_scan_train_load_give_up

template <class Kern>
int launch(Kern kern, int smem, std::atomic<uint64_t>& done, const TrainParams& P, cudaStream_t s) {
    cudaError_t e = ensure_smem(kern, smem, done);
    if (e != cudaSuccess) return cuda_fail(e, "cudaFuncSetAttribute(training scan)");
    const unsigned z = (static_cast<unsigned>(P.nchunks) + kMaxGridY - 1) / kMaxGridY;
    const unsigned y = (static_cast<unsigned>(P.nchunks) + z - 1) / z;
    kern<<<dim3(static_cast<unsigned>(P.nchains), y, z), kNT, smem, s>>>(P);
    e = cudaGetLastError();
    return e == cudaSuccess ? NEED_OK : cuda_fail(e, "training scan launch");
}

template <int FORM, typename T, bool CK, int DT, int CB, bool BWD>
int run_cfg(const TrainParams& P, cudaStream_t s) {
    static std::atomic<uint64_t> done{0};
    constexpr int smem = TrainCfg<FORM, T, CK, DT, CB, BWD>::SMEM;
    if constexpr (BWD) return launch(train_bwd_kernel<FORM, T, CK, DT, CB>, smem, done, P, s);
    else return launch(train_fwd_kernel<FORM, T, CK, DT, CB>, smem, done, P, s);
}

template <bool BWD>
int run(const need_scan_train_args* a, const TrainParams& P, bool narrow, cudaStream_t s) {
    auto form = [&](auto tag) {
        using T = decltype(tag);
        auto go = [&](auto ck) {
            constexpr bool CK = decltype(ck)::value;
            auto width = [&](auto form, auto dt) {
                constexpr int F = decltype(form)::value, DT = decltype(dt)::value;
                if constexpr (!CK)
                    if (narrow) return run_cfg<F, T, CK, DT, 32, BWD>(P, s);
                return run_cfg<F, T, CK, DT, 64, BWD>(P, s);
            };
            constexpr std::integral_constant<int, 0> any{};
            if (a->form == NEED_FORM_GATED) return width(std::integral_constant<int, FORM_GATED>{}, any);
            constexpr std::integral_constant<int, FORM_SSD> ssd{};
            // steps of at most 1/4 (the block's are at most 0.2): e^-r by its series, see exp_neg_small
            if (a->dt_max <= 0.25) return width(ssd, std::integral_constant<int, 1>{});
            return width(ssd, any);
        };
        return a->checkpoint != 0 ? go(std::true_type{}) : go(std::false_type{});
    };
    if (a->dtype == NEED_F32) return form(float{});
    if (a->dtype == NEED_BF16) return form(__nv_bfloat16{});
    return form(__half{});
}

struct Geom {
    int64_t L, CB, ncb, nchains, nchunks, ntiles;
};
// Channels per tile.  64 where the call has enough chains to fill the device;
// 32 (tiles twice as long, where those of 64 are not long already) where it has not: then
// fewer tiles of one chain are in flight and wait for each other's carries, against more
// shuffles in a warp, of which the backward has three times the forward's.  The 8-bit
// forms keep the 64 that share a scale.  The bounds are those of the SSD form in 16 bits;
// device us at 832 channels, 64 / 32 wide, forward and backward:
//   chains of 64      13 (1x16384)              104 (8x2048)              208 (16x1024)
//   SSD bf16     62.7 / 45.2, 86.1 / 82.9   41.8 / 39.1, 74.2 / 77.2   39.3 / 39.0, 73.1 / 77.1
//   SSD f16      63.2 / 45.1, 86.2 / 82.5   41.8 / 38.8, 74.7 / 77.4   39.6 / 38.9, 73.8 / 77.7
//   SSD fp32     110 / 103, 162 / 160       98.6 / 98.4, 154 / 153     99.0 / 98.3, 152 / 152
//   GATED bf16   35.1 / 35.5, 50.2 / 55.7   27.6 / 29.7, 45.2 / 49.9   26.8 / 29.3, 45.2 / 49.7
//   GATED f16    34.7 / 35.4, 49.9 / 55.6   27.3 / 29.9, 45.3 / 50.0   26.6 / 29.6, 45.0 / 49.9
//   GATED fp32   63.2 / 57.7, 100 / 98.0    56.6 / 51.0, 91.2 / 92.4   56.4 / 51.6, 90.1 / 91.4
// So the GATED form in 16 bits, whose 64-wide tiles are the long ones, pays up to a tenth
// for the one rule at 13 to 191 chains (below 8 it gains by it: 4x8192x64 backward 20.3 /
// 16.5), and its fp32 forward a tenth above 191.
Geom geom(int form, int dtype, bool ck, bool bwd, int64_t nb, int64_t T, int64_t C) {
    Geom g;
    g.CB = !ck && nb * ((C + 63) / 64) < (bwd ? 64 : 192) ? 32 : 64;
    g.L = tile_elems(form == NEED_FORM_GATED ? FORM_GATED : FORM_SSD, dtype != NEED_F32, ck, int(g.CB), bwd) / g.CB;
    g.ncb = (C + g.CB - 1) / g.CB;
    g.nchains = nb * g.ncb;
    g.nchunks = (T + g.L - 1) / g.L;
    g.ntiles = g.nchains * g.nchunks;
    return g;
}
// The workspace: header and look-back records, which the call clears, then (SSD
// backward) the partial sums of the gradient of D.
size_t clear_bytes(const Geom& g) {
    return kHdrBytes + (g.nchunks > 1 ? size_t(g.ntiles) * size_t(g.CB) * kRecBytes : 0);
}
size_t ws_size(const Geom& g, int64_t nb, int64_t C, bool dpart) {
    return clear_bytes(g) + (dpart ? size_t(nb) * size_t(g.nchunks) * size_t(C) * 4 : 0);
}

// Whether a [nb, T, C] tensor's rows can be read or written by TMA.
bool tma_rows(const void* ptr, int64_t sb, int64_t st, int es, int64_t nb, int64_t T) {
    auto ok = [&](int64_t n, int64_t s) { return n == 1 || (s > 0 && s * es % 16 == 0 && s * es < (int64_t(1) << 40)); };
    return aligned16(ptr) && ok(T, st) && ok(nb, sb);
}

// Such a tensor (element strides) as a 3-D tensor map with boxes of one warp's rows.
int encode(CUtensorMap* tm, const void* ptr, int64_t sb, int64_t st, int es, CUtensorMapDataType ty, int64_t nb,
           int64_t T, int64_t C, const Geom& g, const char* what) {
    const cuuint64_t row = (C * es + 15) / 16 * 16;  // a size-1 dim's stride is not used
    const cuuint64_t gs[2] = {T > 1 ? cuuint64_t(st * es) : row, nb > 1 ? cuuint64_t(sb * es) : row};
    const cuuint64_t dims[3] = {cuuint64_t(C), cuuint64_t(T), cuuint64_t(nb)};
    const cuuint32_t box[3] = {cuuint32_t(g.CB), cuuint32_t(g.L / kNW), 1}, estr[3] = {1, 1, 1};
    auto fn = encode_fn();
    if (fn == nullptr) return fail(NEED_ERR_CUDA, "cuTensorMapEncodeTiled entry point unavailable");
    const CUresult r = fn(tm, ty, 3, const_cast<void*>(ptr), dims, gs, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                          CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(NEED_ERR_UNSUPPORTED, "cuTensorMapEncodeTiled(%s) failed: %d", what, int(r));
    return NEED_OK;
}

CUtensorMapDataType map_type(int dt) {
    return dt == NEED_F32    ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
           : dt == NEED_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                             : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
}

int prepare(const need_scan_train_args* a, bool bwd, TrainParams* P, Geom* g) {
    if (a == nullptr) return fail(NEED_ERR_INVALID, "args is null");
    if (a->form != NEED_FORM_GATED && a->form != NEED_FORM_SSD)
        return fail(NEED_ERR_INVALID, "form %d: the training scans are GATED and SSD", a->form);
    if (!dtype_ok(a->dtype)) return fail(NEED_ERR_UNSUPPORTED, "dtype %d", a->dtype);
    if (a->checkpoint != 0 && a->checkpoint != 1) return fail(NEED_ERR_INVALID, "checkpoint %d", a->checkpoint);
    if (a->nb < 1 || a->T < 1 || a->C < 1)
        return fail(NEED_ERR_INVALID, "sizes must be >= 1 (nb=%lld T=%lld C=%lld)", (long long)a->nb, (long long)a->T,
                    (long long)a->C);
    const int es = dtype_bytes(a->dtype);
    if (a->nb > INT32_MAX / 8 || a->nb * ((a->T + kSpan - 1) / kSpan) > INT32_MAX / 2 || a->T > INT32_MAX / 2 || a->C > INT32_MAX / 2)
        return fail(NEED_ERR_UNSUPPORTED, "sizes exceed the 32-bit index range");
    *g = geom(a->form, a->dtype, a->checkpoint != 0, bwd, a->nb, a->T, a->C);
    if (g->nchains > INT32_MAX || g->ntiles > INT32_MAX)
        return fail(NEED_ERR_UNSUPPORTED, "too many tiles (%lld)", (long long)g->ntiles);
    const int nin = a->form == NEED_FORM_GATED ? 3 : 5;
    if (a->states == nullptr) return fail(NEED_ERR_INVALID, "states is null");
    if (a->form == NEED_FORM_SSD) {
        if (a->d_skip == nullptr) return fail(NEED_ERR_INVALID, "d_skip is null");
        if (!(a->dt_min >= 0.0) || !(a->dt_max >= a->dt_min) || a->dt_max > 1e30)
            return fail(NEED_ERR_INVALID, "0 <= dt_min <= dt_max <= 1e30 (got %g, %g)", a->dt_min, a->dt_max);
    }
    if (a->checkpoint != 0 && (a->ckpt_values == nullptr || a->ckpt_scales == nullptr))
        return fail(NEED_ERR_INVALID, "the 8-bit checkpoint needs ckpt_values and ckpt_scales");
    if (a->checkpoint != 0 && !aligned16(a->ckpt_values))
        return fail(NEED_ERR_UNSUPPORTED, "ckpt_values is not 16-byte aligned");
    const bool dpart = bwd && a->form == NEED_FORM_SSD;
    if (a->workspace == nullptr || !aligned16(a->workspace))
        return fail(NEED_ERR_WORKSPACE, "workspace is null or not 16-byte aligned");
    if (a->workspace_bytes < ws_size(*g, a->nb, a->C, dpart))
        return fail(NEED_ERR_WORKSPACE, "workspace has %zu bytes, needs %zu", a->workspace_bytes,
                    ws_size(*g, a->nb, a->C, dpart));
    // outputs: rows that TMA can write, at least C long
    auto writable = [&](const void* ptr, int64_t sb, int64_t st) {
        return ptr != nullptr && tma_rows(ptr, sb, st, es, a->nb, a->T) && (a->T == 1 || st >= a->C);
    };
    if (bwd) {
        for (int k = 0; k < nin; ++k)
            if (!writable(a->grad[k], a->grad_stride_b, a->grad_stride_t))
                return fail(NEED_ERR_INVALID, "grad[%d] is null or its rows are not 16-byte aligned, C or more long", k);
        if (a->form == NEED_FORM_SSD && a->grad_d == nullptr) return fail(NEED_ERR_INVALID, "grad_d is null");
    } else if (!writable(a->out, a->out_stride_b, a->out_stride_t)) {
        return fail(NEED_ERR_INVALID, "out is null or its rows are not 16-byte aligned, C or more long");
    }
    const bool stored = bwd && a->checkpoint != 0;
    for (int k = 0; k < nin && !stored; ++k)
        if (a->in[k].ptr == nullptr) return fail(NEED_ERR_INVALID, "in[%d] is null", k);
    if (bwd && a->gout.ptr == nullptr) return fail(NEED_ERR_INVALID, "gout is null");
    if (int rc = ensure_context()) return rc;
    memset(P, 0, sizeof(*P));
    static const char* const names[6] = {"in[0]", "in[1]", "in[2]", "in[3]", "in[4]", "gout"};
    const auto ty = map_type(a->dtype);
    auto stream = [&](int k, const need_view& v, const char* name) {
        if (tma_rows(v.ptr, v.stride_b, v.stride_t, es, a->nb, a->T))
            return encode(&P->tm[k], v.ptr, v.stride_b, v.stride_t, es, ty, a->nb, a->T, a->C, *g, name);
        P->plain |= 1u << k;
        P->src[k] = v.ptr, P->ssb[k] = v.stride_b, P->sst[k] = v.stride_t;
        auto units = [&](int64_t u) {
            return a->C % u == 0 && reinterpret_cast<uintptr_t>(v.ptr) % (u * es) == 0 && (a->T == 1 || v.stride_t % u == 0) &&
                   (a->nb == 1 || v.stride_b % u == 0);
        };
        P->unit[k] = es == 2 && units(4) ? 4 : units(2) ? 2 : 1;
        return int(NEED_OK);
    };
    for (int k = 0; k < nin; ++k) {
        const int64_t pitch = (a->C + kGroup - 1) / kGroup * kGroup;
        // the 8-bit values of every stream as one [nin * nb, T, ncb * 64] tensor: the
        // kernel adds its stream's first sequence to b
        const int rc = stored ? encode(&P->tm[k], a->ckpt_values, a->T * pitch, pitch, 1, CU_TENSOR_MAP_DATA_TYPE_UINT8,
                                       nin * a->nb, a->T, pitch, *g, "ckpt_values")
                              : stream(k, a->in[k], names[k]);
        if (rc) return rc;
    }
    if (bwd)
        if (int rc = stream(nin, a->gout, names[5])) return rc;
    for (int k = 0; k < (bwd ? nin : 1); ++k)
        if (int rc = bwd ? encode(&P->tmo[k], a->grad[k], a->grad_stride_b, a->grad_stride_t, es, ty, a->nb, a->T, a->C,
                                  *g, "grad")
                         : encode(&P->tmo[0], a->out, a->out_stride_b, a->out_stride_t, es, ty, a->nb, a->T, a->C, *g,
                                  "out"))
            return rc;
    P->nb = int32_t(a->nb);
    P->T = int32_t(a->T);
    P->C = int32_t(a->C);
    P->ncb = int32_t(g->ncb);
    P->nchains = int32_t(g->nchains);
    P->nchunks = int32_t(g->nchunks);
    P->ngroups = int32_t((a->C + kGroup - 1) / kGroup);
    P->nspans = int32_t((a->T + kSpan - 1) / kSpan);
    // few chains have many of their tiles in flight at once: look further back
    P->depth = g->nchains < 64 ? kDeep : kNear;
    P->dskip = a->d_skip;
    P->dt_min = static_cast<float>(a->dt_min);
    P->dt_scale = static_cast<float>(a->dt_max - a->dt_min);
    P->h0 = a->h0;
    P->h_final = a->h_final;
    P->seg = a->seg_start;
    P->sgb = a->seg_stride_b;
    P->sgt = a->seg_stride_t;
    P->states = a->states;
    P->q = a->ckpt_values;
    P->qs = a->ckpt_scales;
    P->g_final = a->g_final;
    P->grad_h0 = a->grad_h0;
    unsigned char* ws = static_cast<unsigned char*>(a->workspace);
    P->hdr = reinterpret_cast<uint32_t*>(ws);
    P->agg = reinterpret_cast<unsigned long long*>(ws + kHdrBytes);
    P->incl = reinterpret_cast<uint32_t*>(ws + kHdrBytes + size_t(g->ntiles) * size_t(g->CB) * 8);
    P->dpart = reinterpret_cast<float*>(ws + clear_bytes(*g));
    P->polls = lookback_polls();
    P->load_polls = g_load_give_up.load(std::memory_order_relaxed) ? 0 : kTmaPolls;
    return NEED_OK;
}

int clear_records(const need_scan_train_args* a, const Geom& g, cudaStream_t s) {
    const cudaError_t e = cudaMemsetAsync(a->workspace, 0, clear_bytes(g), s);
    return e == cudaSuccess ? NEED_OK : cuda_fail(e, "cudaMemsetAsync(training scan records)");
}

}  // namespace

extern "C" {

int64_t need_scan_train_chunk_len(void) { return kSpan; }

int64_t need_scan_train_group(void) { return kGroup; }

size_t need_scan_train_workspace_size(int32_t form, int32_t dtype, int32_t checkpoint, int32_t backward, int64_t nb,
                                      int64_t T, int64_t C) {
    if (nb < 1 || T < 1 || C < 1) return kHdrBytes;
    return ws_size(geom(form, dtype, checkpoint != 0, backward != 0, nb, T, C), nb, C, backward != 0 && form == NEED_FORM_SSD);
}

int need_scan_train_error(uint32_t* error_out, need_stream_t stream) {
    if (error_out == nullptr) return fail(NEED_ERR_INVALID, "null argument");
    void* word = nullptr;
    cudaError_t e = cudaGetSymbolAddress(&word, g_train_error);
    if (e == cudaSuccess) e = cudaMemcpyAsync(error_out, word, 4, cudaMemcpyDeviceToHost, stream);
    if (e == cudaSuccess) e = cudaStreamSynchronize(stream);
    if (e == cudaSuccess && *error_out != 0) e = cudaMemsetAsync(word, 0, 4, stream);
    if (e != cudaSuccess) return cuda_fail(e, "need_scan_train_error");
    return ok();
}

void need_test_scan_train_load_give_up(int32_t on) { g_load_give_up.store(on != 0, std::memory_order_relaxed); }

int need_scan_train_forward(const need_scan_train_args* args, need_stream_t stream) {
    TrainParams P;
    Geom g;
    if (int rc = prepare(args, false, &P, &g)) return rc;
    if (int rc = clear_records(args, g, stream)) return rc;
    if (int rc = run<false>(args, P, g.CB == 32, stream)) return rc;
    return ok();
}

int need_scan_train_backward(const need_scan_train_args* args, need_stream_t stream) {
    TrainParams P;
    Geom g;
    if (int rc = prepare(args, true, &P, &g)) return rc;
    if (int rc = clear_records(args, g, stream)) return rc;
    if (int rc = run<true>(args, P, g.CB == 32, stream)) return rc;
    if (args->form == NEED_FORM_SSD)
        if (int rc = column_sums(P.dpart, args->nb * g.nchunks, args->C, args->grad_d, stream)) return rc;
    return ok();
}

}  // extern "C"
