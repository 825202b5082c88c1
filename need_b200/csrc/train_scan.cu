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
// Tiles are 64 tokens x 64 channels, one CTA each: 8 row warps of 8 rows, a
// lane owning one pair of channels (packed fp32 arithmetic), and a look-back
// warp.  The forward writes the fp32 state entering each tile ([nb, chunks,
// C], 1/32 of one 16-bit stream); the backward runs its tile's states again
// from there, so it reads neither h nor any gate from memory, and both
// directions stream their algorithmic bytes once: 8 and 14 B per element
// (GATED, 16 bit), 12 and 22 B (SSD).
//
// Across tiles the carry travels as in scan_kernel.cuh (single pass, decoupled
// look-back over the kTrainDepth tiles before and the inclusive carry of the
// one before those, composed in that fixed order, so results are
// bit-reproducible), but with its own records: 32-bit words holding the
// complement of a float's bits, 0 while unwritten.  The call clears them on
// its stream before the launch, so a workspace carries nothing from one call
// to the next: captured graphs may share one, or be replayed in any order.
// Every wait is bounded; a tile that gives up sets the workspace's error word
// and passes NaN on.
//
// Checkpoints in 8 bits: the forward also writes its inputs as e4m3 with one
// power of two per token and 64 channels, and the backward reads those (5 + 2
// bytes per SSD element in place of 12) -- the gradient is then the formula's
// at the stored values, from the true state entering each tile.
#include <cuda_fp8.h>
#include <string.h>

#include <algorithm>

#include "host_common.h"
#include "need_scan.h"
#include "scan_kernel.cuh"
#include "train_common.cuh"

using namespace need;

namespace {

constexpr int kL = 64, kCB = 64;      // tokens and channels per tile
constexpr int kNW = 8, kR = kL / kNW;  // row warps and rows per warp
constexpr int kNT = (kNW + 1) * 32;    // threads: the row warps and the look-back warp
constexpr int kTrainDepth = 3;         // tile maps composed before an inclusive carry
constexpr int kHdrBytes = WS_HDR_WORDS * 4;
constexpr int kTileRecBytes = kCB * 12;  // per tile: (A, B) and the inclusive carry of each channel

struct TrainParams {
    CUtensorMap tm[6];  // the streamed inputs, and gout (backward, last)
    int32_t nb, T, C, ncb, nchains, nchunks;
    const float* dskip;
    float dt_min, dt_scale;
    const float* h0;       // forward: initial state; backward: unused (the states hold it)
    float* h_final;        // forward
    const uint8_t* seg;
    int64_t sgb, sgt;
    float* states;         // [nb, nchunks, C] the state entering each tile
    void* out;             // forward
    int64_t osb, ost;
    uint8_t* q;            // 8-bit values [nin][nb][T][ncb * 64]
    uint8_t* qs;           // their scales [nin][nb][T][ncb]
    void* grad[5];         // backward: [nb, T, C] each, in in[] order
    const float* g_final;  // backward: gradient of the final state or null
    float* grad_h0;        // backward, optional
    float* dpart;          // backward SSD: [nb * nchunks, C] partial sums of the gradient of D
    uint32_t* hdr;
    ulonglong2* agg;           // [ntiles][32] (A, B) of the lane's two channels
    unsigned long long* incl;  // [ntiles][32] the carry past the tile, two channels
    uint32_t polls;
};

// ------------------------------------------------------------------ maps
// Affine maps c -> A c + B with A == 0 meaning "drops c", whatever c holds.
__device__ __forceinline__ float2 apply(float2 A, float2 c, float2 B) {
    const float2 r = ffma2(A, c, B);
    return make_float2(A.x == 0.0f ? B.x : r.x, A.y == 0.0f ? B.y : r.y);
}
__device__ __forceinline__ float2 mulz(float2 a, float2 b) {
    const float2 r = fmul2(a, b);
    return make_float2(a.x == 0.0f || b.x == 0.0f ? 0.0f : r.x, a.y == 0.0f || b.y == 0.0f ? 0.0f : r.y);
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

// ------------------------------------------------------------------ inputs
// A lane's channel pair of row r of a 16- or 32-bit slot.
template <typename T>
__device__ __forceinline__ float2 pair_at(const unsigned char* slot, int r, int lane) {
    return widen(reinterpret_cast<const typename Ops<T>::P*>(slot)[r * (kCB / 2) + lane]);
}
// The same of an 8-bit slot, times its row's scale.
__device__ __forceinline__ float2 pair8_at(const unsigned char* slot, int r, int lane, float scale) {
    const __nv_fp8x2_storage_t q = reinterpret_cast<const __nv_fp8x2_storage_t*>(slot)[r * (kCB / 2) + lane];
    const float2 f = __half22float2(static_cast<__half2>(__nv_cvt_fp8x2_to_halfraw2(q, __NV_E4M3)));
    return make_float2(f.x * scale, f.y * scale);
}

template <int FORM, typename T, bool CK, bool BWD>
struct TrainCfg {
    static constexpr int NIN = FORM == FORM_GATED ? 3 : 5;
    static constexpr int IN_BYTES = (BWD && CK) ? 1 : Ops<T>::BYTES;     // per streamed input element
    static constexpr int IN_SLOT = kL * kCB * IN_BYTES;
    static constexpr int OFF_GOUT = NIN * IN_SLOT;
    static constexpr int OFF_MAP = OFF_GOUT + (BWD ? kL * kCB * Ops<T>::BYTES : 0);  // [NW][32] (A, B) float4
    static constexpr int OFF_FWD = OFF_MAP + kNW * 32 * 16;                // BWD: [NW][32] forward B, float2
    static constexpr int OFF_IN = OFF_FWD + (BWD ? kNW * 32 * 8 : 0);      // [NW][32] carry entering each warp
    static constexpr int OFF_HIN = OFF_IN + kNW * 32 * 8;                  // BWD: [NW][32] state entering each warp
    static constexpr int OFF_SCALE = OFF_HIN + (BWD ? kNW * 32 * 8 : 0);   // BWD CK: [NW][NIN][R] fp32 scales
    static constexpr int OFF_BAR = OFF_SCALE + (BWD && CK ? kNW * NIN * kR * 4 : 0);
    static constexpr int SMEM = OFF_BAR + (kNW + 1) * 8 + 128;
};

// ------------------------------------------------------------------ look-back
// The look-back warp's work for one tile: composes the tile's map from the
// warps' maps, publishes it, takes the carry that enters the tile, publishes
// the one that leaves it, and leaves in s_in the carry entering each warp's
// rows.  `order(w)` gives the w-th warp met by the carry; `carry` holds the
// initial value when `first`, else it is read.  Returns the carry past the tile.
template <bool REV, class Wait>
__device__ __forceinline__ float2 look_back(const TrainParams& p, int64_t tile, int pos, bool last, int lane,
                                            float2& carry, const float4* s_map, float2* s_in, Wait maps_ready) {
    const int nagg = min(pos - 1, kTrainDepth);
    bool have = pos == 0, mapped = false;
    float2 A, B;
    for (uint32_t it = 0;; ++it) {
        bool progressed = false;
        if (!have) {
            bool valid = true;
            float2 accA = splat2(1.0f), accB = splat2(0.0f);
            for (int j = 0; j < nagg; ++j) {
                const ulonglong2 m = ld_relaxed_v2u64(p.agg + (tile - int64_t(j + 1) * p.nchains) * 32 + lane);
                valid &= rec_set(m.x) & rec_set(m.y);  // (A0, B0), (A1, B1)
                accB = apply(accA, make_float2(rec_hi(m.x), rec_hi(m.y)), accB);
                accA = mulz(accA, make_float2(rec_lo(m.x), rec_lo(m.y)));
            }
            const unsigned long long c = ld_relaxed_u64(p.incl + (tile - int64_t(nagg + 1) * p.nchains) * 32 + lane);
            valid &= rec_set(c);
            if (__all_sync(0xffffffffu, valid)) {
                carry = apply(accA, make_float2(rec_lo(c), rec_hi(c)), accB);
                have = progressed = true;
            }
        }
        // with the carry in, nothing else is polled: suspend on the barrier
        if (!mapped && maps_ready(have)) {
            A = splat2(1.0f);
            B = splat2(0.0f);
#pragma unroll
            for (int k = 0; k < kNW; ++k) {  // in the order the carry meets the warps
                const float4 m = s_map[(REV ? kNW - 1 - k : k) * 32 + lane];
                B = apply(make_float2(m.x, m.y), B, make_float2(m.z, m.w));
                A = mulz(make_float2(m.x, m.y), A);
            }
            if (!last && pos > 0)  // the first tile's map is never composed: its carry is known
                st_relaxed_v2u64(p.agg + tile * 32 + lane, rec_pair(A.x, B.x), rec_pair(A.y, B.y));
            mapped = progressed = true;
        }
        if (mapped && have) break;
        if (!have && it >= p.polls) {  // go on without a predecessor's carry
            if (lane == 0) atomicOr(&p.hdr[WS_ERROR], ERR_LOOKBACK);
            carry = splat2(__int_as_float(0x7fc00000));
            have = true;
        } else if (have && it - min(it, p.polls) >= kTmaPolls) {  // the row warps' own waits are shorter
            if (lane == 0) atomicOr(&p.hdr[WS_ERROR], ERR_TMA);
            A = splat2(0.0f);
            B = splat2(__int_as_float(0x7fc00000));
            break;
        }
        if (!progressed && !have && it >= 2) __nanosleep(64);
    }
    const float2 past = apply(A, carry, B);
    if (!last) {
        st_relaxed_u64(p.incl + tile * 32 + lane, rec_pair(past.x, past.y));
    }
    float2 c = carry;
#pragma unroll
    for (int k = 0; k < kNW; ++k) {
        const int w = REV ? kNW - 1 - k : k;
        s_in[w * 32 + lane] = c;
        const float4 m = s_map[w * 32 + lane];
        c = apply(make_float2(m.x, m.y), c, make_float2(m.z, m.w));
    }
    return past;
}

// This lane's two channels of a [.., C] fp32 row (0 past C).
__device__ __forceinline__ float2 ld_pair(const float* row, int c, int C) {
    return make_float2(c < C ? row[c] : 0.0f, c + 1 < C ? row[c + 1] : 0.0f);
}
__device__ __forceinline__ void st_pair(float* row, int c, int C, float2 v) {
    if (c < C) row[c] = v.x;
    if (c + 1 < C) row[c + 1] = v.y;
}

struct Tile {
    int pos, chunk, cblk, b, t0, c0, nvalid;
    int64_t tile;
};
__device__ __forceinline__ Tile tile_of(const TrainParams& p, bool rev) {
    Tile t;
    t.tile = blockIdx.x;
    t.pos = static_cast<int>(blockIdx.x) / p.nchains;  // in the order the carry meets the tiles
    const int chain = static_cast<int>(blockIdx.x) - t.pos * p.nchains;
    t.chunk = rev ? p.nchunks - 1 - t.pos : t.pos;
    t.b = chain / p.ncb;
    t.cblk = chain - t.b * p.ncb;
    t.t0 = t.chunk * kL;
    t.c0 = t.cblk * kCB;
    t.nvalid = min(kL, p.T - t.t0);
    return t;
}

// Bit j: row wr0 + j of the tile starts a segment (rows past T: clear).
__device__ __forceinline__ uint32_t reset_bits(const TrainParams& p, const Tile& tl, int wr0, int lane) {
    bool r = false;
    const int t = tl.t0 + wr0 + lane;
    if (p.seg != nullptr && lane < kR && t < p.T) r = p.seg[tl.b * p.sgb + int64_t(t) * p.sgt] != 0;
    return __ballot_sync(0xffffffffu, r);
}

// ------------------------------------------------------------------ gates
// a, 1 - a and w = s(gate) * value from a row's streams.
template <int FORM, typename T>
__device__ __forceinline__ void decay(const TrainParams& p, float2 x0, float2& a, float2& na) {
    if constexpr (FORM == FORM_GATED) {
        sig_pair<T>(x0, a, na);
    } else {
        float2 s, n;
        sig_pair<T>(x0, s, n);
        const float2 rate = ffma2(s, splat2(p.dt_scale), splat2(p.dt_min));
        exp_neg<T>(rate, a, na);
    }
}

// ------------------------------------------------------------------ forward
template <int FORM, typename T, bool CK>
__global__ void __launch_bounds__(kNT) train_fwd_kernel(const __grid_constant__ TrainParams p) {
    using K = TrainCfg<FORM, T, CK, false>;
    using O = Ops<T>;
    extern __shared__ unsigned char smem_raw[];
    unsigned char* base =
        reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 127) & ~uintptr_t(127));
    float4* s_map = reinterpret_cast<float4*>(base + K::OFF_MAP);
    float2* s_in = reinterpret_cast<float2*>(base + K::OFF_IN);
    uint64_t* s_bar = reinterpret_cast<uint64_t*>(base + K::OFF_BAR);
    uint64_t* s_maps = s_bar + kNW;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const Tile tl = tile_of(p, false);
    if (threadIdx.x == 0) {
        for (int w = 0; w < kNW; ++w) mbar_init(&s_bar[w], 1);
        mbar_init(s_maps, kNW * 32);
        fence_barrier_init();
    }
    __syncthreads();
    const int c = tl.c0 + 2 * lane;  // this lane's channels c, c + 1

    if (warp == kNW) {
        const bool last = tl.chunk + 1 == p.nchunks;
        float2 carry = splat2(0.0f);
        if (tl.pos == 0 && p.h0 != nullptr) carry = ld_pair(p.h0 + int64_t(tl.b) * p.C, c, p.C);
        const float2 past = look_back<false>(p, tl.tile, tl.pos, last, lane, carry, s_map, s_in, [&](bool block) {
            return __all_sync(0xffffffffu, block ? mbar_try_wait(s_maps, 0) : mbar_test_wait(s_maps, 0));
        });
        __syncwarp();
        named_arrive(1, kNT);
        st_pair(p.states + (int64_t(tl.b) * p.nchunks + tl.chunk) * p.C, c, p.C, carry);
        if (last && p.h_final != nullptr) st_pair(p.h_final + int64_t(tl.b) * p.C, c, p.C, past);
        return;
    }

    const int wr0 = warp * kR;
    const int rows = max(0, min(kR, tl.nvalid - wr0));
    if (lane == 0 && rows > 0) {
        mbar_arrive_expect_tx(&s_bar[warp], K::NIN * K::IN_SLOT / kNW);
#pragma unroll
        for (int k = 0; k < K::NIN; ++k)
            tma_load_3d(base + k * K::IN_SLOT + wr0 * kCB * K::IN_BYTES, &p.tm[k], tl.c0, tl.t0 + wr0, tl.b,
                        &s_bar[warp]);
    }
    const uint32_t resets = reset_bits(p, tl, wr0, lane);
    float2 D = splat2(0.0f);
    if constexpr (FORM == FORM_SSD) D = ld_pair(p.dskip, c, p.C);
    if (rows > 0 && !mbar_wait_bounded(&s_bar[warp], 0, kTmaPolls)) {
        atomicOr(&p.hdr[WS_ERROR], ERR_TMA);
        mbar_wait_bounded(&s_bar[warp], 0, kTmaPolls);
    }
    const unsigned char* in[K::NIN];
#pragma unroll
    for (int k = 0; k < K::NIN; ++k) in[k] = base + k * K::IN_SLOT + wr0 * kCB * K::IN_BYTES;

    // phase 1: each row's state from a zero entering state (H) and the product
    // of a up to it (P); the last is the warp's map
    float2 P[kR], H[kR];
    float2 A = splat2(1.0f), B = splat2(0.0f);
    if (rows > 0) {
#pragma unroll
        for (int j = 0; j < kR; ++j) {
            float2 a, na, s, n;
            decay<FORM, T>(p, pair_at<T>(in[0], j, lane), a, na);
            sig_pair<T>(pair_at<T>(in[1], j, lane), s, n);
            const float2 b = fmul2(na, fmul2(s, pair_at<T>(in[2], j, lane)));
            if ((resets >> j) & 1u) {
                A = splat2(0.0f);
                B = b;
            } else if (j < rows) {
                B = ffma2(a, B, b);
                A = (resets & ((1u << j) - 1u)) ? A : fmul2(a, A);  // stays 0 after a reset
            }
            P[j] = A;
            H[j] = B;
        }
    }
    s_map[warp * 32 + lane] = make_float4(A.x, A.y, B.x, B.y);
    mbar_arrive(s_maps);

    if constexpr (CK) {  // the 8-bit copies, while the carry comes in
        const int64_t pitch = int64_t(p.ncb) * kCB;
#pragma unroll
        for (int k = 0; k < K::NIN; ++k) {
#pragma unroll
            for (int j = 0; j < kR; ++j) {
                if (j < rows) {
                    const float2 x = pair_at<T>(in[k], j, lane);
                    const uint32_t top =
                        __reduce_max_sync(0xffffffffu, max(__float_as_uint(x.x) & 0x7fffffffu,
                                                           __float_as_uint(x.y) & 0x7fffffffu));
                    const uint32_t sc = e4m3_scale_byte(top);
                    const int64_t row = (int64_t(k) * p.nb + tl.b) * p.T + tl.t0 + wr0 + j;
                    *reinterpret_cast<uint16_t*>(p.q + row * pitch + c) = e4m3_pair(x, sc);
                    if (lane == 0) p.qs[row * p.ncb + tl.cblk] = static_cast<uint8_t>(sc);
                }
            }
        }
    }
    named_sync(1, kNT);

    // phase 2: the states from the entering one, and the outputs
    const float2 hin = s_in[warp * 32 + lane];
    T* orow = static_cast<T*>(p.out) + tl.b * p.osb + int64_t(tl.t0 + wr0) * p.ost + c;
#pragma unroll
    for (int j = 0; j < kR; ++j) {
        if (j < rows) {
            const bool cut = (resets & ((2u << j) - 1u)) != 0u;
            float2 o = cut ? H[j] : ffma2(P[j], hin, H[j]);
            if constexpr (FORM == FORM_SSD) {
                float2 s, n, g;
                sig_pair<T>(pair_at<T>(in[3], j, lane), s, n);
                sig_pair<T>(pair_at<T>(in[4], j, lane), g, n);
                o = fmul2(ffma2(s, o, fmul2(D, pair_at<T>(in[2], j, lane))), g);
            }
            if (c < p.C) *reinterpret_cast<typename O::P*>(orow + j * p.ost) = O::pack(o.x, o.y);
        }
    }
}

// ------------------------------------------------------------------ backward
template <int FORM, typename T, bool CK>
__global__ void __launch_bounds__(kNT) train_bwd_kernel(const __grid_constant__ TrainParams p) {
    using K = TrainCfg<FORM, T, CK, true>;
    using O = Ops<T>;
    extern __shared__ unsigned char smem_raw[];
    unsigned char* base =
        reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 127) & ~uintptr_t(127));
    float4* s_map = reinterpret_cast<float4*>(base + K::OFF_MAP);
    float2* s_fwd = reinterpret_cast<float2*>(base + K::OFF_FWD);
    float2* s_in = reinterpret_cast<float2*>(base + K::OFF_IN);
    float2* s_hin = reinterpret_cast<float2*>(base + K::OFF_HIN);
    float* s_scale = reinterpret_cast<float*>(base + K::OFF_SCALE);
    uint64_t* s_bar = reinterpret_cast<uint64_t*>(base + K::OFF_BAR);
    uint64_t* s_maps = s_bar + kNW;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const Tile tl = tile_of(p, true);
    if (threadIdx.x == 0) {
        for (int w = 0; w < kNW; ++w) mbar_init(&s_bar[w], 1);
        mbar_init(s_maps, kNW * 32);
        fence_barrier_init();
    }
    __syncthreads();
    const int c = tl.c0 + 2 * lane;

    if (warp == kNW) {
        const bool last = tl.chunk == 0;
        float2 h = ld_pair(p.states + (int64_t(tl.b) * p.nchunks + tl.chunk) * p.C, c, p.C);
        float2 carry = splat2(0.0f);
        if (tl.pos == 0 && p.g_final != nullptr) carry = ld_pair(p.g_final + int64_t(tl.b) * p.C, c, p.C);
        bool handed = false;
        const float2 past = look_back<true>(p, tl.tile, tl.pos, last, lane, carry, s_map, s_in, [&](bool block) {
            const bool ready =
                __all_sync(0xffffffffu, block ? mbar_try_wait(s_maps, 0) : mbar_test_wait(s_maps, 0));
            if (ready) {  // the states entering the warps first: they wait for no other tile
                handed = true;
#pragma unroll
                for (int w = 0; w < kNW; ++w) {
                    s_hin[w * 32 + lane] = h;
                    const float4 m = s_map[w * 32 + lane];
                    h = apply(make_float2(m.x, m.y), h, s_fwd[w * 32 + lane]);
                }
                __syncwarp();
                named_arrive(1, kNT);
            }
            return ready;
        });
        if (!handed) named_arrive(1, kNT);  // gave up: the row warps are let go
        __syncwarp();
        named_arrive(2, kNT);
        if (last && p.grad_h0 != nullptr) st_pair(p.grad_h0 + int64_t(tl.b) * p.C, c, p.C, past);
        return;
    }

    const int wr0 = warp * kR;
    const int rows = max(0, min(kR, tl.nvalid - wr0));
    if (lane == 0 && rows > 0) {
        mbar_arrive_expect_tx(&s_bar[warp], (K::NIN * K::IN_SLOT + kL * kCB * O::BYTES) / kNW);
#pragma unroll
        for (int k = 0; k < K::NIN; ++k)
            tma_load_3d(base + k * K::IN_SLOT + wr0 * kCB * K::IN_BYTES, &p.tm[k], tl.c0, tl.t0 + wr0,
                        CK ? k * p.nb + tl.b : tl.b, &s_bar[warp]);
        tma_load_3d(base + K::OFF_GOUT + wr0 * kCB * O::BYTES, &p.tm[K::NIN], tl.c0, tl.t0 + wr0, tl.b,
                    &s_bar[warp]);
    }
    const uint32_t resets = reset_bits(p, tl, wr0, lane);
    if constexpr (CK) {
        for (int i = lane; i < K::NIN * kR; i += 32) {
            const int k = i / kR, j = i - k * kR;
            float f = 0.0f;
            if (j < rows)
                f = e4m3_scale(p.qs[((int64_t(k) * p.nb + tl.b) * p.T + tl.t0 + wr0 + j) * p.ncb + tl.cblk]);
            s_scale[warp * K::NIN * kR + i] = f;
        }
        __syncwarp();
    }
    float2 D = splat2(0.0f);
    if constexpr (FORM == FORM_SSD) D = ld_pair(p.dskip, c, p.C);
    if (rows > 0 && !mbar_wait_bounded(&s_bar[warp], 0, kTmaPolls)) {
        atomicOr(&p.hdr[WS_ERROR], ERR_TMA);
        mbar_wait_bounded(&s_bar[warp], 0, kTmaPolls);
    }
    auto input = [&](int k, int j) {
        const unsigned char* slot = base + k * K::IN_SLOT + wr0 * kCB * K::IN_BYTES;
        if constexpr (CK) return pair8_at(slot, j, lane, s_scale[(warp * K::NIN + k) * kR + j]);
        else return pair_at<T>(slot, j, lane);
    };
    auto gout = [&](int j) { return pair_at<T>(base + K::OFF_GOUT + wr0 * kCB * O::BYTES, j, lane); };

    // phase 1: the warp's maps.  Forward: h_out = A h_in + B.  Backward, over
    // the same a: mu_first = A mu_in + M, M = sum over rows of (product of a up
    // to the row) e.
    float2 a[kR], h[kR];
    float2 A = splat2(1.0f), B = splat2(0.0f), M = splat2(0.0f);
    if (rows > 0) {
#pragma unroll
        for (int j = 0; j < kR; ++j) {
            float2 na, s, n;
            decay<FORM, T>(p, input(0, j), a[j], na);
            sig_pair<T>(input(1, j), s, n);
            const float2 b = fmul2(na, fmul2(s, input(2, j)));
            float2 e = gout(j);
            if constexpr (FORM == FORM_SSD) {
                float2 sc, so;
                sig_pair<T>(input(3, j), sc, n);
                sig_pair<T>(input(4, j), so, n);
                e = fmul2(e, fmul2(so, sc));
            }
            h[j] = b;
            if ((resets >> j) & 1u) {
                A = splat2(0.0f);
                B = b;
            } else if (j < rows) {
                B = ffma2(a[j], B, b);
                if ((resets & ((1u << j) - 1u)) == 0u) {
                    A = fmul2(a[j], A);
                    M = ffma2(A, e, M);
                }
            }
        }
    }
    s_map[warp * 32 + lane] = make_float4(A.x, A.y, M.x, M.y);
    s_fwd[warp * 32 + lane] = B;
    mbar_arrive(s_maps);
    named_sync(1, kNT);

    // the states of the warp's rows, from the one entering them
    const float2 hin = s_hin[warp * 32 + lane];
    if (rows > 0) {
        float2 hp = hin;
#pragma unroll
        for (int j = 0; j < kR; ++j) {
            h[j] = ((resets >> j) & 1u) ? h[j] : ffma2(a[j], hp, h[j]);
            hp = h[j];
        }
    }
    named_sync(2, kNT);

    // phase 2: the rows from last to first
    float2 mu = s_in[warp * 32 + lane];
    float2 dD = splat2(0.0f);
    const int64_t row0 = (int64_t(tl.b) * p.T + tl.t0 + wr0) * p.C + c;
    auto put = [&](int k, int j, float2 v) {
        if (c < p.C)
            *reinterpret_cast<typename O::P*>(static_cast<T*>(p.grad[k]) + row0 + int64_t(j) * p.C) =
                O::pack(v.x, v.y);
    };
#pragma unroll
    for (int j = kR - 1; j >= 0; --j) {
        if (j < rows) {
            const bool reset = ((resets >> j) & 1u) != 0u;
            const float2 prev = reset ? splat2(0.0f) : (j > 0 ? h[j > 0 ? j - 1 : 0] : hin);
            float2 s0, n0, aj, na, sg, ng;
            const float2 x0 = input(0, j), val = input(2, j);
            if constexpr (FORM == FORM_GATED) {
                sig_pair<T>(x0, aj, na);
            } else {
                sig_pair<T>(x0, s0, n0);
                exp_neg<T>(ffma2(s0, splat2(p.dt_scale), splat2(p.dt_min)), aj, na);
            }
            sig_pair<T>(input(1, j), sg, ng);
            const float2 go = gout(j);
            float2 e = go, gs = go;
            if constexpr (FORM == FORM_SSD) {
                float2 sc, nc, so, no;
                sig_pair<T>(input(3, j), sc, nc);
                sig_pair<T>(input(4, j), so, no);
                gs = fmul2(go, so);
                e = fmul2(gs, sc);
                put(3, j, fmul2(fmul2(gs, h[j]), fmul2(sc, nc)));
                const float2 v = ffma2(sc, h[j], fmul2(D, val));
                put(4, j, fmul2(fmul2(gs, v), no));
                dD = ffma2(gs, val, dD);
            }
            const float2 lam = fadd2(e, mu);
            mu = reset ? splat2(0.0f) : fmul2(aj, lam);
            const float2 w = fmul2(sg, val);
            const float2 da = fmul2(lam, fadd2(prev, make_float2(-w.x, -w.y)));
            const float2 dw = fmul2(lam, na);
            if constexpr (FORM == FORM_GATED) {
                put(0, j, fmul2(da, fmul2(aj, na)));
                put(2, j, fmul2(dw, sg));
            } else {
                const float2 slope = fmul2(fmul2(s0, n0), splat2(-p.dt_scale));
                put(0, j, fmul2(fmul2(da, aj), slope));
                put(2, j, ffma2(dw, sg, fmul2(D, gs)));
            }
            put(1, j, fmul2(fmul2(dw, val), fmul2(sg, ng)));
        }
    }
    if constexpr (FORM == FORM_SSD) {
        // the tile's sum for the gradient of D: the warps' sums in a fixed order
        s_fwd[warp * 32 + lane] = dD;  // the look-back warp is done with it
        named_sync(3, kNW * 32);
        if (warp == 0) {
            float2 sum = splat2(0.0f);
#pragma unroll
            for (int w = 0; w < kNW; ++w) sum = fadd2(sum, s_fwd[w * 32 + lane]);
            st_pair(p.dpart + (int64_t(tl.b) * p.nchunks + tl.chunk) * p.C, c, p.C, sum);
        }
    }
}

// ------------------------------------------------------------------ launch
template <class Kern>
int launch(Kern kern, int smem, std::atomic<uint64_t>& done, const TrainParams& P, int64_t ntiles, cudaStream_t s) {
    cudaError_t e = ensure_smem(kern, smem, done);
    if (e != cudaSuccess) return cuda_fail(e, "cudaFuncSetAttribute(training scan)");
    kern<<<static_cast<unsigned>(ntiles), kNT, smem, s>>>(P);
    e = cudaGetLastError();
    return e == cudaSuccess ? NEED_OK : cuda_fail(e, "training scan launch");
}

template <int FORM, typename T, bool CK, bool BWD>
int run_cfg(const TrainParams& P, int64_t ntiles, cudaStream_t s) {
    static std::atomic<uint64_t> done{0};
    constexpr int smem = TrainCfg<FORM, T, CK, BWD>::SMEM;
    if constexpr (BWD) return launch(train_bwd_kernel<FORM, T, CK>, smem, done, P, ntiles, s);
    else return launch(train_fwd_kernel<FORM, T, CK>, smem, done, P, ntiles, s);
}

template <bool BWD>
int run(const need_scan_train_args* a, const TrainParams& P, int64_t ntiles, cudaStream_t s) {
    auto form = [&](auto tag) {
        using T = decltype(tag);
        const bool ck = a->checkpoint != 0;
        if (a->form == NEED_FORM_GATED)
            return ck ? run_cfg<FORM_GATED, T, true, BWD>(P, ntiles, s) : run_cfg<FORM_GATED, T, false, BWD>(P, ntiles, s);
        return ck ? run_cfg<FORM_SSD, T, true, BWD>(P, ntiles, s) : run_cfg<FORM_SSD, T, false, BWD>(P, ntiles, s);
    };
    if (a->dtype == NEED_F32) return form(float{});
    if (a->dtype == NEED_BF16) return form(__nv_bfloat16{});
    return form(__half{});
}

struct Geom {
    int64_t ncb, nchains, nchunks, ntiles;
};
Geom geom(int64_t nb, int64_t T, int64_t C) {
    Geom g;
    g.ncb = (C + kCB - 1) / kCB;
    g.nchains = nb * g.ncb;
    g.nchunks = (T + kL - 1) / kL;
    g.ntiles = g.nchains * g.nchunks;
    return g;
}
size_t rec_bytes(const Geom& g) { return g.nchunks > 1 ? size_t(g.ntiles) * kTileRecBytes : 0; }
size_t ws_size(const Geom& g, int64_t nb, int64_t C, bool dpart) {
    return kHdrBytes + rec_bytes(g) + (dpart ? size_t(nb) * size_t(g.nchunks) * size_t(C) * 4 : 0);
}

// A [nb, T, C] tensor (element strides) as a 3-D tensor map with boxes of one
// warp's rows.
int encode(CUtensorMap* tm, const void* ptr, int64_t sb, int64_t st, int es, CUtensorMapDataType ty, int64_t nb,
           int64_t T, int64_t C, const char* what) {
    if (ptr == nullptr) return fail(NEED_ERR_INVALID, "%s is null", what);
    if (!aligned16(ptr)) return fail(NEED_ERR_UNSUPPORTED, "%s is not 16-byte aligned", what);
    const int64_t sizes[2] = {T, nb}, strides[2] = {st, sb};
    cuuint64_t gs[2];
    int64_t prev = ((C * es + 15) / 16) * 16;  // a size-1 dim's stride is not used
    for (int i = 0; i < 2; ++i) {
        int64_t by = prev;
        if (sizes[i] > 1) {
            by = strides[i] * es;
            if (strides[i] <= 0 || by % 16 != 0 || by >= (int64_t(1) << 40))
                return fail(NEED_ERR_UNSUPPORTED, "%s: stride %lld must be positive and a multiple of 16 bytes", what,
                            (long long)strides[i]);
        }
        gs[i] = static_cast<cuuint64_t>(by);
        prev = by * sizes[i];
        if (prev >= (int64_t(1) << 40)) prev = 16;
    }
    const cuuint64_t dims[3] = {cuuint64_t(C), cuuint64_t(T), cuuint64_t(nb)};
    const cuuint32_t box[3] = {kCB, kR, 1}, estr[3] = {1, 1, 1};
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
    const int es = dtype_bytes(a->dtype), group = 16 / es;
    if (a->C % group != 0)
        return fail(NEED_ERR_UNSUPPORTED, "C=%lld must be a multiple of %d for this dtype", (long long)a->C, group);
    if (a->nb > INT32_MAX / 8 || a->T > INT32_MAX / 2 || a->C > INT32_MAX / 2)
        return fail(NEED_ERR_UNSUPPORTED, "sizes exceed the 32-bit index range");
    *g = geom(a->nb, a->T, a->C);
    if (g->nchains > INT32_MAX || g->ntiles > INT32_MAX)
        return fail(NEED_ERR_UNSUPPORTED, "too many tiles (%lld)", (long long)g->ntiles);
    const int nin = a->form == NEED_FORM_GATED ? 3 : 5;
    if (a->states == nullptr) return fail(NEED_ERR_INVALID, "states is null");
    if (a->form == NEED_FORM_SSD) {
        if (a->d_skip == nullptr) return fail(NEED_ERR_INVALID, "d_skip is null");
        if (!(a->dt_min >= 0.0) || !(a->dt_max >= a->dt_min))
            return fail(NEED_ERR_INVALID, "0 <= dt_min <= dt_max (got %g, %g)", a->dt_min, a->dt_max);
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
    if (bwd) {
        for (int k = 0; k < nin; ++k)
            if (a->grad[k] == nullptr || !aligned16(a->grad[k]))
                return fail(NEED_ERR_INVALID, "grad[%d] is null or not 16-byte aligned", k);
        if (a->form == NEED_FORM_SSD && a->grad_d == nullptr) return fail(NEED_ERR_INVALID, "grad_d is null");
    } else {
        if (a->out == nullptr || !aligned16(a->out)) return fail(NEED_ERR_INVALID, "out is null or not 16-byte aligned");
        if ((a->T > 1 && (a->out_stride_t < a->C || a->out_stride_t % group != 0)) ||
            (a->nb > 1 && (a->out_stride_b <= 0 || a->out_stride_b % group != 0)))
            return fail(NEED_ERR_UNSUPPORTED, "out strides must be positive multiples of %d elements", group);
    }
    if (int rc = ensure_context()) return rc;
    memset(P, 0, sizeof(*P));
    static const char* const names[5] = {"in[0]", "in[1]", "in[2]", "in[3]", "in[4]"};
    if (bwd && a->checkpoint != 0) {
        // every stream's 8-bit values as one [nin * nb, T, ncb * 64] tensor: the
        // kernel adds its stream's first row of sequences to b
        const int64_t pitch = g->ncb * kCB;
        for (int k = 0; k < nin; ++k)
            if (int rc = encode(&P->tm[k], a->ckpt_values, a->T * pitch, pitch, 1, CU_TENSOR_MAP_DATA_TYPE_UINT8,
                                nin * a->nb, a->T, pitch, "ckpt_values"))
                return rc;
    } else {
        for (int k = 0; k < nin; ++k)
            if (int rc = encode(&P->tm[k], a->in[k].ptr, a->in[k].stride_b, a->in[k].stride_t, es, map_type(a->dtype),
                                a->nb, a->T, a->C, names[k]))
                return rc;
    }
    if (bwd)
        if (int rc = encode(&P->tm[nin], a->gout.ptr, a->gout.stride_b, a->gout.stride_t, es, map_type(a->dtype), a->nb,
                            a->T, a->C, "gout"))
            return rc;
    P->nb = int32_t(a->nb);
    P->T = int32_t(a->T);
    P->C = int32_t(a->C);
    P->ncb = int32_t(g->ncb);
    P->nchains = int32_t(g->nchains);
    P->nchunks = int32_t(g->nchunks);
    P->dskip = a->d_skip;
    P->dt_min = static_cast<float>(a->dt_min);
    P->dt_scale = static_cast<float>(a->dt_max - a->dt_min);
    P->h0 = a->h0;
    P->h_final = a->h_final;
    P->seg = a->seg_start;
    P->sgb = a->seg_stride_b;
    P->sgt = a->seg_stride_t;
    P->states = a->states;
    P->out = a->out;
    P->osb = a->out_stride_b;
    P->ost = a->out_stride_t;
    P->q = a->ckpt_values;
    P->qs = a->ckpt_scales;
    for (int k = 0; k < nin; ++k) P->grad[k] = a->grad[k];
    P->g_final = a->g_final;
    P->grad_h0 = a->grad_h0;
    unsigned char* ws = static_cast<unsigned char*>(a->workspace);
    P->hdr = reinterpret_cast<uint32_t*>(ws);
    P->agg = reinterpret_cast<ulonglong2*>(ws + kHdrBytes);
    P->incl = reinterpret_cast<unsigned long long*>(ws + kHdrBytes + size_t(g->ntiles) * kCB * 8);
    P->dpart = reinterpret_cast<float*>(ws + kHdrBytes + rec_bytes(*g));
    P->polls = lookback_polls();
    return NEED_OK;
}

int clear_records(const need_scan_train_args* a, const Geom& g, cudaStream_t s) {
    const cudaError_t e = cudaMemsetAsync(a->workspace, 0, kHdrBytes + rec_bytes(g), s);
    return e == cudaSuccess ? NEED_OK : cuda_fail(e, "cudaMemsetAsync(training scan records)");
}

}  // namespace

extern "C" {

int64_t need_scan_train_chunk_len(void) { return kL; }

int64_t need_scan_train_group(void) { return kCB; }

size_t need_scan_train_workspace_size(int32_t form, int32_t backward, int64_t nb, int64_t T, int64_t C) {
    if (nb < 1 || T < 1 || C < 1) return kHdrBytes;
    return ws_size(geom(nb, T, C), nb, C, backward != 0 && form == NEED_FORM_SSD);
}

int need_scan_train_forward(const need_scan_train_args* args, need_stream_t stream) {
    TrainParams P;
    Geom g;
    if (int rc = prepare(args, false, &P, &g)) return rc;
    if (int rc = clear_records(args, g, stream)) return rc;
    if (int rc = run<false>(args, P, g.ntiles, stream)) return rc;
    return ok();
}

int need_scan_train_backward(const need_scan_train_args* args, need_stream_t stream) {
    TrainParams P;
    Geom g;
    if (int rc = prepare(args, true, &P, &g)) return rc;
    if (int rc = clear_records(args, g, stream)) return rc;
    if (int rc = run<true>(args, P, g.ntiles, stream)) return rc;
    if (args->form == NEED_FORM_SSD)
        if (int rc = column_sums(P.dpart, args->nb * g.nchunks, args->C, args->grad_d, stream)) return rc;
    return ok();
}

}  // extern "C"
