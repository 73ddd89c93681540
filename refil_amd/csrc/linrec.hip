// Gated linear recurrence over an episode, forward / backward / one acting step (include/refil_hip.h: refil_linrec_*).
//
//   L_t = c softplus(decay) sigmoid(ga_t),  a_t = exp(-L_t)
//   h_t = [no reset at t] a_t h_{t-1} + sqrt(1 - a_t^2) sigmoid(gi_t) x_t,   y_t = h_t
//
// The gates do not read h, so a step is the affine map h -> A h + H and maps compose: (A2, H2) o (A1, H1) = (A2 A1, A2 H1 + H2). Time is
// cut three times: a thread composes S consecutive steps, a wave its 64 / TC time-threads by shuffles, a workgroup its four waves through
// LDS; the carry goes from tile to tile (16 to 64 steps) in registers. A reset cuts the chain: it travels beside the map as a flag instead of as
// A = 0, so that a NaN or Inf in front of it does not pass (0 * NaN).
//
// Backward: with g_t the whole gradient of h_t, g_t = dy_t + c_t and c_{t-1} = a_t g_t [no reset at t] -- the same maps A in reverse
// order, R_t in H_t's place. h_{t-1} is computed again from the fp32 state that the forward keeps at every tile's start (one value per
// 16 to 64 steps), not read from the rounded y: no 16-bit rounding enters the gradient, and 7 streams move where reading y would make 8.
// The gate gradients come without a division by sqrt(1 - a^2):
//   q_t = d loss / d log L_t = g_t (sigmoid(gi) x a^2 L / sqrt(1 - a^2) - a h_{t-1} L),   L / sqrt(1 - a^2) -> sqrt(L / 2) -> 0
//   dga_t = q_t (1 - sigmoid(ga)),   ddecay = sum q_t sigmoid(decay) / softplus(decay)
//
// Bound by memory and by the latency of a tile (gates, shuffles, one barrier), which other waves of the compute unit hide. 96 ragged
// episodes of 81 steps, 1024 channels in fp32: 30 + 45 us. Where sequences are too few to fill the card, time is cut into chunks, one round
// of workgroups in all: a first launch makes the chunks' maps (3 streams read; backward 2), the second starts every chunk from the maps in
// front of it. 4 sequences of 8192 steps, 1024 channels in bf16: 42 + 58 us forward, 28 + 101 us backward (maps and outputs; 4.6 .. 4.9 TB/s).
#include <type_traits>

#include "kernels.h"
#include "profile.h"
#include "vecio.h"

namespace refil {

struct LinrecK {
    const void* x; const void* ga; const void* gi; long x_sB, x_sT, ga_sB, ga_sT, gi_sB, gi_sT;
    const float* decay; float scale;
    const float* h0; const uint8_t* reset; long rs_sB, rs_sT; const int* lengths;
    void* y; long y_sB, y_sT; float* h_last; float* saved;
    const void* dy; long dy_sB, dy_sT; const float* dh_last;
    void* dx; void* dga; void* dgi; long d_sB, d_sT; float* dh0; float* part;
    int B, T, C, D, ch, ncol, nchunk, tiles_per_chunk, ntile;      // ch: channels of a workgroup (64, or 256 for few 16-bit sequences)
    float* sumA; float* sumH;          // [B][nchunk][C]: the maps of whole chunks (A = -1: the chunk holds a reset)
};

constexpr int LR_V = 4, LR_WAVES = 4;
// TC lanes of a wave lie along the channels (4 each), the other 64 / TC along time. 64: a wave reads 256 neighbouring channels at a time and
// needs no scan of its own; 16, for narrow rows: 64 channels, four time-threads joined by shuffles.
// Steps of a thread: what joins a tile costs the same whatever S is, registers grow with it. fp32 (16 bytes a value and stream) is bound by
// occupancy -- 96 episodes of 81 steps, 1024 channels: 31 + 46 us at S 2, 37 + 64 at S 4 -- 16-bit types by instructions.
template <class T, int TC> struct LrGeo {
    static constexpr int CH = TC * LR_V, TW = 64 / TC, S = sizeof(T) == 4 ? 2 : 4, TT = LR_WAVES * TW * S;
};
// Which: 64 lanes where 16 would have their time axis cut anyway (lr_plan: two chunks or more fit while (episode, 64 channels) pairs are at most
// half of 768), so that the cheaper tile wins; beyond, 16 lanes pass once over the data. bf16, forward + backward at 33.5 million elements, 64 against
// 16 lanes: 64 pairs (B 4, T 8192, C 1024) 100 + 133 against 102 + 141 us, 128 pairs 96 + 129 / 101 + 143, 256 pairs 96 + 130 / 97 + 143, 384 pairs
// (36.9 million) 109 + 155 / 116 + 162; 512 pairs 96 + 130 / 63 + 118, 1024 pairs 93 + 130 / 67 + 127. fp32 does not gain (78 + 116 against
// 78 + 120 us at B 4, T 4096, C 1024).
static int lr_tc(int dtype, int B, int C) { return dtype != REFIL_F32 && C > 128 && (long)B * cdiv(C, 64) <= 384 ? 64 : 16; }
static int lr_tile(int dtype, int B, int C) {
    return dtype == REFIL_F32 ? LrGeo<float, 16>::TT : lr_tc(dtype, B, C) == 64 ? LrGeo<bf16_t, 64>::TT : LrGeo<bf16_t, 16>::TT;
}

__device__ __forceinline__ float softplus_(float v) { return fmaxf(v, 0.f) + log1pf(expf(-fabsf(v))); }

struct LrGate { float sa, si, L, a, beta, lob; };      // lob = L / sqrt(1 - a^2)
// 1 - a^2 = 1 - exp(-2L) = 2 a sinh(L): below L = 0.35 by sinh's series (next term L^9 / 362880: 6e-10 of it), where the difference would
// lose digits. WIDE = false: no channel's L reaches 0.35.
template <bool WIDE, bool BWD>
__device__ __forceinline__ LrGate lr_gate(float ga, float gi, float rate) {
    LrGate g;
    g.sa = fast_sigmoid(ga); g.si = fast_sigmoid(gi);
    g.L = rate * g.sa;
    g.a = fast_exp(-g.L);
    const float q = g.L * g.L;
    float om = (g.a * (g.L + g.L)) * fmaf(q, fmaf(q, fmaf(q, 1.98412698e-4f, 8.33333333e-3f), 1.66666667e-1f), 1.0f);
    if (WIDE) om = g.L < 0.35f ? om : fmaf(-g.a, g.a, 1.0f);
    if (BWD) {
        const float rs = __builtin_amdgcn_rsqf(fmaxf(om, 1e-37f));
        g.beta = om * rs;
        g.lob = g.L * rs;
    } else g.beta = __builtin_amdgcn_sqrtf(om);
    return g;
}

// rates of the workgroup's channels, one softplus each (the caller issues its first loads in front of the barrier)
__device__ __forceinline__ void lr_rates(const LinrecK& k, int ch0, int channels, float* s_rate) {
    if ((int)threadIdx.x < channels) {
        const int c = ch0 + (int)threadIdx.x;
        s_rate[threadIdx.x] = c < k.C ? k.scale * softplus_(k.decay[c % k.D]) : 0.f;
    }
    lds_barrier();
}

// S steps of one stream from `base` (the episode's first step, channel c0). `whole` (wave-uniform): every step is live and every channel
// there. Otherwise a lane reads from where it may -- a step before the episode's end, V channels inside the row -- and puts right what it
// got: no branches, one wait (B 3, T 5001, 997 channels of fp16: 73 against 99 us; the wave has a live step, so the episode has one). fp32,
// whose registers are full, and rows of fewer than V channels branch instead.
template <class T, int S>
__device__ __forceinline__ void lr_load(Raw<T, LR_V> (&r)[S], const T* base, long sT, int t0, int Tb, int c0, int C, bool whole, unsigned absent = 0u) {
    if (whole) {
        const T* p = base + (long)t0 * sT;
#pragma unroll
        for (int s = 0; s < S; ++s) { r[s] = ld_raw<T, LR_V>(p, LR_V); p += sT; }
    } else if (sizeof(T) == 2 && C >= LR_V) {
        const int back = max(c0 - (C - LR_V), 0);
        const T* p = base - back;
#pragma unroll
        for (int s = 0; s < S; ++s) r[s] = ld_raw<T, LR_V>(p + (long)min(t0 + s, Tb - 1) * sT, LR_V);
        if (C % LR_V) {
#pragma unroll
            for (int s = 0; s < S; ++s) r[s] = raw_down<T, LR_V>(r[s], min(back, LR_V - 1));
        }
#pragma unroll
        for (int s = 0; s < S; ++s)
#pragma unroll
            for (int w = 0; w < (int)(sizeof(r[s].w) / 4); ++w) r[s].w[w] = t0 + s < Tb ? r[s].w[w] : absent;
    } else {
#pragma unroll
        for (int s = 0; s < S; ++s) r[s] = ld_raw<T, LR_V>(base + (long)(t0 + s) * sT, t0 + s < Tb ? C - c0 : 0, absent);
    }
}
// the reset flags of S steps: loaded with the data, looked at when the maps are built
template <bool RST, int S>
__device__ __forceinline__ void lr_load_cuts(uint8_t (&r)[S], const LinrecK& k, int b, int t0, int Tb) {
    if (RST) {
        const uint8_t* p = k.reset + (long)b * k.rs_sB;
#pragma unroll
        for (int s = 0; s < S; ++s) r[s] = p[(long)min(t0 + s, Tb - 1) * k.rs_sT];      // (the wave has a live step: Tb >= 1)
    }
}
template <bool RST, int S>
__device__ __forceinline__ int lr_cuts(const uint8_t (&r)[S], int t0, int Tb) {
    int cuts = 0;
    if (RST) {
#pragma unroll
        for (int s = 0; s < S; ++s) cuts |= (t0 + s < Tb && r[s] ? 1 : 0) << s;
    }
    return cuts;
}

// The maps of the n chunks in front (behind): chunk first + i * step is the i-th to apply. Each of the 16 time-threads composes a run of
// them, the wave joins its four by shuffles; the waves' maps go to LDS (the caller's next barrier orders them).
template <int TC> struct LrFront { float A[LR_WAVES][TC * LR_V], H[LR_WAVES][TC * LR_V]; int cut[LR_WAVES]; };
template <int TC>
__device__ __forceinline__ void lr_front(const LinrecK& k, LrFront<TC>& f, int b, int c0, int cl, int nv, int wave, int tw, int n, int first, int step) {
    constexpr int TW = 64 / TC, AT = 4;
    float A[LR_V], H[LR_V]; int cut = 0;
#pragma unroll
    for (int i = 0; i < LR_V; ++i) { A[i] = 1.f; H[i] = 0.f; }
    const int per = cdiv(n, LR_WAVES * TW), i0 = (wave * TW + tw) * per, i1 = min(i0 + per, n);
    for (int j = i0; j < i1; j += AT) {           // (AT chunks' loads at a time)
        Raw<float> a[AT], h[AT];
#pragma unroll
        for (int q = 0; q < AT; ++q) {
            const long o = ((long)b * k.nchunk + first + min(j + q, i1 - 1) * step) * k.C + c0;
            a[q] = ld_raw<float>(k.sumA + o, nv); h[q] = ld_raw<float>(k.sumH + o, nv);
        }
#pragma unroll
        for (int q = 0; q < AT; ++q) {
            const bool in = j + q < i1, c = in && nv > 0 && raw_get(a[q], 0) < 0.f;               // (a reset cuts every channel)
            cut |= (int)c;
#pragma unroll
            for (int i = 0; i < LR_V; ++i) {
                const float av = in ? raw_get(a[q], i) : 1.f, hv = in ? raw_get(h[q], i) : 0.f;
                H[i] = c ? hv : fmaf(av, H[i], hv);
                A[i] *= av;
            }
        }
    }
    if constexpr (TW > 1) {
#pragma unroll
        for (int d = 1; d < TW; d *= 2) {
            const int pc = __shfl_up(cut, d * TC);
#pragma unroll
            for (int i = 0; i < LR_V; ++i) {
                const float pA = __shfl_up(A[i], d * TC), pH = __shfl_up(H[i], d * TC);
                if (tw >= d) { H[i] = cut ? H[i] : fmaf(A[i], pH, H[i]); A[i] *= pA; }
            }
            if (tw >= d) cut |= pc;
        }
    }
    if (tw == TW - 1) {
#pragma unroll
        for (int i = 0; i < LR_V; ++i) { f.A[wave][cl + i] = A[i]; f.H[wave][cl + i] = H[i]; }
        if (cl == 0) f.cut[wave] = cut;
    }
}
template <int TC>
__device__ __forceinline__ void lr_front_apply(const LrFront<TC>& f, int cl, float (&carry)[LR_V]) {
#pragma unroll
    for (int w = 0; w < LR_WAVES; ++w) {
        const int c = f.cut[w];
#pragma unroll
        for (int i = 0; i < LR_V; ++i) carry[i] = c ? f.H[w][cl + i] : fmaf(f.A[w][cl + i], carry[i], f.H[w][cl + i]);
    }
}

// One workgroup per (episode, CH channels, chunk of the time axis). FINAL: the outputs, starting from the carry of the chunks in front;
// else the chunk's whole map only. Steps past the episode's end are not loaded: their decay gate is -inf (a = 1, no input), the state
// stays. A wave whose steps all lie there skips the arithmetic. The next tile's loads are in flight from the moment this tile's gates are
// computed: over its scans, barrier and stores.
template <class T, int TC, bool FINAL, bool RST>
__global__ void __launch_bounds__(256, sizeof(T) == 4 ? 4 : 3) linrec_fwd(const LinrecK k) {
    typedef LrGeo<T, TC> G;
    constexpr int V = LR_V, TW = G::TW, S = G::S, TT = G::TT, CH = G::CH;
    __shared__ float s_rate[CH];
    __shared__ float sA[2][LR_WAVES][CH], sH[2][LR_WAVES][CH];
    __shared__ int sCut[2][LR_WAVES];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int b = (int)(blockIdx.x / k.ncol), ch0 = (int)(blockIdx.x % k.ncol) * CH, chunk = blockIdx.y;
    const int cl = (lane % TC) * V, c0 = ch0 + cl, nv = min(max(k.C - c0, 0), V);
    const int tw = lane / TC;
    const bool all_ch = ch0 + CH <= k.C;
    const int Tb = k.lengths ? min(max(k.lengths[b], 0), k.T) : k.T;
    const T* xb = (const T*)k.x + (long)b * k.x_sB + c0;
    const T* gab = (const T*)k.ga + (long)b * k.ga_sB + c0;
    const T* gib = (const T*)k.gi + (long)b * k.gi_sB + c0;
    const int tile0 = chunk * k.tiles_per_chunk, tile1 = min(tile0 + k.tiles_per_chunk, k.ntile);
    Raw<T, V> rx[S], rga[S], rgi[S];
    uint8_t rc[S];
    auto load = [&](int tile) {
        const int w0 = tile * TT + wave * (TW * S), t0 = w0 + tw * S;
        if (tile < tile1 && w0 < Tb) {
            const bool whole = all_ch && w0 + TW * S <= Tb;
            lr_load(rga, gab, k.ga_sT, t0, Tb, c0, k.C, whole, NEG_INF_WORD<T>);
            lr_load(rgi, gib, k.gi_sT, t0, Tb, c0, k.C, whole);
            lr_load(rx, xb, k.x_sT, t0, Tb, c0, k.C, whole);
            lr_load_cuts<RST, S>(rc, k, b, t0, Tb);
        }
    };
    load(tile0);
    float carry[V];
#pragma unroll
    for (int i = 0; i < V; ++i) carry[i] = FINAL && k.h0 && i < nv ? k.h0[(long)b * k.C + c0 + i] : 0.f;
    __shared__ LrFront<TC> front;
    if (FINAL && chunk > 0) lr_front(k, front, b, c0, cl, nv, wave, tw, chunk, 0, 1);
    lr_rates(k, ch0, CH, s_rate);
    if (FINAL && chunk > 0) lr_front_apply(front, cl, carry);
    float rate[V], top = 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i) { rate[i] = s_rate[cl + i]; top = fmaxf(top, rate[i]); }
    const bool wide = __any(!(top < 0.35f));
    float cA[V]; int ccut = 0;       // !FINAL: the chunk's map so far (its H is `carry`, started from zero)
#pragma unroll
    for (int i = 0; i < V; ++i) cA[i] = 1.f;
    for (int tile = tile0; tile < tile1; ++tile) {
        const int p = tile & 1, tw0 = tile * TT + wave * (TW * S), t0 = tw0 + tw * S;
        const bool any_live = tw0 < Tb;                                   // (wave-uniform)
        float a[S][V], u[S][V], A[V], H[V], eA[V], eH[V];
        int cuts = 0, cut = 0, ecut = 0;
#pragma unroll
        for (int i = 0; i < V; ++i) { A[i] = 1.f; H[i] = 0.f; eA[i] = 1.f; eH[i] = 0.f; }
        if (any_live) {
            cuts = lr_cuts<RST, S>(rc, t0, Tb);
            cut = cuts != 0;
            auto gates = [&](auto w) {
#pragma unroll
                for (int s = 0; s < S; ++s)
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        const LrGate g = lr_gate<decltype(w)::value, false>(raw_get(rga[s], i), raw_get(rgi[s], i), rate[i]);
                        a[s][i] = g.a;
                        u[s][i] = g.beta * (g.si * raw_get(rx[s], i));
                    }
            };
            if (wide) gates(std::true_type{}); else gates(std::false_type{});
        }
        load(tile + 1);
        if (any_live) {
#pragma unroll
            for (int s = 0; s < S; ++s)
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    H[i] = RST && (cuts >> s & 1) ? u[s][i] : fmaf(a[s][i], H[i], u[s][i]);
                    A[i] *= a[s][i];
                }
            // inclusive over the wave's time-threads, then exclusive
            if constexpr (TW > 1) {
#pragma unroll
            for (int d = 1; d < TW; d *= 2) {
                const int pc = RST ? __shfl_up(cut, d * TC) : 0;
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const float pA = __shfl_up(A[i], d * TC), pH = __shfl_up(H[i], d * TC);
                    if (tw >= d) { H[i] = RST && cut ? H[i] : fmaf(A[i], pH, H[i]); A[i] *= pA; }
                }
                if (tw >= d) cut |= pc;
            }
            if (RST) ecut = __shfl_up(cut, TC);
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float pA = __shfl_up(A[i], TC), pH = __shfl_up(H[i], TC);
                eA[i] = tw ? pA : 1.f; eH[i] = tw ? pH : 0.f;
            }
            if (tw == 0) ecut = 0;
            }
        }
        if (tw == TW - 1) {
#pragma unroll
            for (int i = 0; i < V; ++i) { sA[p][wave][cl + i] = A[i]; sH[p][wave][cl + i] = H[i]; }
            if (RST && lane % TC == 0) sCut[p][wave] = cut;
        }
        lds_barrier();
        float h[V];
        if (FINAL && k.saved && wave == 0 && tw == 0) {
            float* o = k.saved + ((long)b * k.ntile + tile) * k.C + c0;
#pragma unroll
            for (int i = 0; i < V; ++i)
                if (i < nv) o[i] = carry[i];
        }
#pragma unroll
        for (int w = 0; w < LR_WAVES; ++w) {
            const int wc = RST ? sCut[p][w] : 0;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                if (w == wave) h[i] = carry[i];
                const float wA = sA[p][w][cl + i], wH = sH[p][w][cl + i];
                carry[i] = wc ? wH : fmaf(wA, carry[i], wH);
                if (!FINAL) cA[i] *= wA;
            }
            ccut |= wc;
        }
        if (FINAL && tw0 < k.T) {
            T* yp = (T*)k.y + (long)b * k.y_sB + (long)t0 * k.y_sT + c0;
            if (TW > 1 && any_live) {
#pragma unroll
                for (int i = 0; i < V; ++i) h[i] = ecut ? eH[i] : fmaf(eA[i], h[i], eH[i]);
            }
#pragma unroll
            for (int s = 0; s < S; ++s) {
                const int t = t0 + s;
                float o[V];
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    if (any_live) h[i] = RST && (cuts >> s & 1) ? u[s][i] : fmaf(a[s][i], h[i], u[s][i]);
                    o[i] = t < Tb ? h[i] : 0.f;
                }
                if (t < k.T) st_raw<T, V>(yp, raw_pack<T, V>(o), nv);
                yp += k.y_sT;
            }
        }
    }
    if (wave == 0 && tw == 0) {
        if (!FINAL) {
            const long o = ((long)b * k.nchunk + chunk) * k.C + c0;
#pragma unroll
            for (int i = 0; i < V; ++i)
                if (i < nv) { k.sumA[o + i] = ccut ? -1.f : cA[i]; k.sumH[o + i] = carry[i]; }
        } else if (k.h_last && chunk == k.nchunk - 1) {
#pragma unroll
            for (int i = 0; i < V; ++i)
                if (i < nv) k.h_last[(long)b * k.C + c0 + i] = carry[i];
        }
    }
}

// the same cut of the time axis in reverse order
template <class T, int TC, bool FINAL, bool RST>
__global__ void __launch_bounds__(256, sizeof(T) == 4 || !FINAL ? 3 : 2) linrec_bwd(const LinrecK k) {
    typedef LrGeo<T, TC> G;
    constexpr int V = LR_V, TW = G::TW, S = G::S, TT = G::TT, CH = G::CH;
    __shared__ float s_rate[CH];
    __shared__ float sA[2][LR_WAVES][CH], sH[2][LR_WAVES][CH], sR[2][LR_WAVES][CH];
    __shared__ int sCut[2][LR_WAVES];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int b = (int)(blockIdx.x / k.ncol), ch0 = (int)(blockIdx.x % k.ncol) * CH, chunk = blockIdx.y;
    const int cl = (lane % TC) * V, c0 = ch0 + cl, nv = min(max(k.C - c0, 0), V);
    const int tw = lane / TC;
    const bool all_ch = ch0 + CH <= k.C;
    const int Tb = k.lengths ? min(max(k.lengths[b], 0), k.T) : k.T;
    const T* xb = (const T*)k.x + (long)b * k.x_sB + c0;
    const T* gab = (const T*)k.ga + (long)b * k.ga_sB + c0;
    const T* gib = (const T*)k.gi + (long)b * k.gi_sB + c0;
    const T* dyb = (const T*)k.dy + (long)b * k.dy_sB + c0;
    const int tile0 = chunk * k.tiles_per_chunk, tile1 = min(tile0 + k.tiles_per_chunk, k.ntile);
    Raw<T, V> rx[S], rdy[S], rga[S], rgi[S];
    uint8_t rc[S];
    float hin[V];
    auto load = [&](int tile) {
        const int w0 = tile * TT + wave * (TW * S), t0 = w0 + tw * S;
        if (tile >= tile0 && w0 < Tb) {
            const bool whole = all_ch && w0 + TW * S <= Tb;
            lr_load(rga, gab, k.ga_sT, t0, Tb, c0, k.C, whole, NEG_INF_WORD<T>);
            lr_load(rdy, dyb, k.dy_sT, t0, Tb, c0, k.C, whole);
            if (FINAL) {
                lr_load(rgi, gib, k.gi_sT, t0, Tb, c0, k.C, whole);
                lr_load(rx, xb, k.x_sT, t0, Tb, c0, k.C, whole);
                const float* o = k.saved + ((long)b * k.ntile + tile) * k.C + c0;
#pragma unroll
                for (int i = 0; i < V; ++i) hin[i] = i < nv ? o[i] : 0.f;
            }
            lr_load_cuts<RST, S>(rc, k, b, t0, Tb);
        }
    };
    load(tile1 - 1);
    float carry[V], cA[V], dl[V]; int ccut = 0;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        carry[i] = FINAL && k.dh_last && i < nv ? k.dh_last[(long)b * k.C + c0 + i] : 0.f;
        cA[i] = 1.f; dl[i] = 0.f;
    }
    __shared__ LrFront<TC> front;
    const int behind = k.nchunk - 1 - chunk;
    if (FINAL && behind > 0) lr_front(k, front, b, c0, cl, nv, wave, tw, behind, k.nchunk - 1, -1);
    lr_rates(k, ch0, CH, s_rate);
    if (FINAL && behind > 0) lr_front_apply(front, cl, carry);
    float rate[V], top = 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i) { rate[i] = s_rate[cl + i]; top = fmaxf(top, rate[i]); }
    const bool wide = __any(!(top < 0.35f));
    for (int tile = tile1 - 1; tile >= tile0; --tile) {
        const int p = tile & 1, tw0 = tile * TT + wave * (TW * S), t0 = tw0 + tw * S;
        const bool any_live = tw0 < Tb;
        // what the outputs need of an element: a, sigmoid(ga), f = sqrt(1 - a^2) sigmoid(gi), w = sigmoid(gi) x a L / sqrt(1 - a^2) and
        // xd = x (1 - sigmoid(gi)):  dx = g f,  dgi = dx xd,  q = g a (w - h_{t-1} L)
        float a[S][V], sa[S][V], f[S][V], w_[S][V], xd[S][V];
        float A[V], H[V], R[V], B[V], eA[V], eH[V], xA[V], xR[V];
        int cuts = 0, fcut = 0, rcut = 0, ecut = 0, xcut = 0;
#pragma unroll
        for (int i = 0; i < V; ++i) { A[i] = B[i] = 1.f; H[i] = R[i] = 0.f; eA[i] = xA[i] = 1.f; eH[i] = xR[i] = 0.f; }
        if (any_live) {
            cuts = lr_cuts<RST, S>(rc, t0, Tb);
            fcut = rcut = cuts != 0;
            auto gates = [&](auto w) {
#pragma unroll
                for (int s = 0; s < S; ++s)
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        if (FINAL) {
                            const LrGate g = lr_gate<decltype(w)::value, true>(raw_get(rga[s], i), raw_get(rgi[s], i), rate[i]);
                            const float x = raw_get(rx[s], i), sx = g.si * x;
                            a[s][i] = g.a; sa[s][i] = g.sa; f[s][i] = g.beta * g.si; w_[s][i] = sx * (g.a * g.lob); xd[s][i] = x - sx;
                        } else a[s][i] = fast_exp(-rate[i] * fast_sigmoid(raw_get(rga[s], i)));
                    }
            };
            if (FINAL && wide) gates(std::true_type{}); else gates(std::false_type{});
#pragma unroll
            for (int s = 0; s < S; ++s)
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    if (FINAL) {
                        const float u = f[s][i] * raw_get(rx[s], i);
                        H[i] = RST && (cuts >> s & 1) ? u : fmaf(a[s][i], H[i], u);
                    }
                    A[i] *= a[s][i];
                }
#pragma unroll
            for (int s = S - 1; s >= 0; --s)
#pragma unroll
                for (int i = 0; i < V; ++i) R[i] = RST && (cuts >> s & 1) ? 0.f : a[s][i] * (raw_get(rdy[s], i) + R[i]);
        }
        if (!FINAL) load(tile - 1);
        if (any_live) {
            // forward: inclusive prefix of (A, H); backward: inclusive suffix of (B, R)
#pragma unroll
            for (int i = 0; i < V; ++i) B[i] = A[i];
            if constexpr (TW > 1) {
#pragma unroll
            for (int d = 1; d < TW; d *= 2) {
                const int pc = RST ? __shfl_up(fcut, d * TC) : 0, nc = RST ? __shfl_down(rcut, d * TC) : 0;
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    if (FINAL) {
                        const float pA = __shfl_up(A[i], d * TC), pH = __shfl_up(H[i], d * TC);
                        if (tw >= d) { H[i] = RST && fcut ? H[i] : fmaf(A[i], pH, H[i]); A[i] *= pA; }
                    }
                    const float nA = __shfl_down(B[i], d * TC), nR = __shfl_down(R[i], d * TC);
                    if (tw + d < TW) { R[i] = RST && rcut ? R[i] : fmaf(B[i], nR, R[i]); B[i] *= nA; }
                }
                if (tw >= d) fcut |= pc;
                if (tw + d < TW) rcut |= nc;
            }
            if (FINAL) {
                if (RST) { ecut = __shfl_up(fcut, TC); xcut = __shfl_down(rcut, TC); }
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const float pA = __shfl_up(A[i], TC), pH = __shfl_up(H[i], TC), nA = __shfl_down(B[i], TC), nR = __shfl_down(R[i], TC);
                    eA[i] = tw ? pA : 1.f; eH[i] = tw ? pH : 0.f;
                    xA[i] = tw < TW - 1 ? nA : 1.f; xR[i] = tw < TW - 1 ? nR : 0.f;
                }
                if (tw == 0) ecut = 0;
                if (tw == TW - 1) xcut = 0;
            }
            }
        }
        if (tw == 0) {
#pragma unroll
            for (int i = 0; i < V; ++i) { sA[p][wave][cl + i] = B[i]; sR[p][wave][cl + i] = R[i]; }
            if (RST && lane % TC == 0) sCut[p][wave] = rcut;
        }
        if (FINAL && tw == TW - 1) {
#pragma unroll
            for (int i = 0; i < V; ++i) sH[p][wave][cl + i] = H[i];
        }
        lds_barrier();
        float c[V];
#pragma unroll
        for (int w = LR_WAVES - 1; w >= 0; --w) {
            const int wc = RST ? sCut[p][w] : 0;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                if (w == wave) c[i] = carry[i];
                const float wA = sA[p][w][cl + i], wR = sR[p][w][cl + i];
                carry[i] = wc ? wR : fmaf(wA, carry[i], wR);
                if (!FINAL) cA[i] *= wA;
            }
            ccut |= wc;
        }
        if (FINAL && tw0 < k.T) {
            const long o = (long)b * k.d_sB + (long)t0 * k.d_sT + c0;
            T* xp = (T*)k.dx + o; T* ap = (T*)k.dga + o; T* ip = (T*)k.dgi + o;
            if (any_live) {
#pragma unroll
                for (int w = 0; w < LR_WAVES - 1; ++w) {
                    if (w < wave) {
                        const int wc = RST ? sCut[p][w] : 0;
#pragma unroll
                        for (int i = 0; i < V; ++i) hin[i] = wc ? sH[p][w][cl + i] : fmaf(sA[p][w][cl + i], hin[i], sH[p][w][cl + i]);
                    }
                }
                if constexpr (TW > 1) {
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        hin[i] = ecut ? eH[i] : fmaf(eA[i], hin[i], eH[i]);
                        c[i] = xcut ? xR[i] : fmaf(xA[i], c[i], xR[i]);
                    }
                }
#pragma unroll
                for (int s = 0; s < S; ++s)
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        const float u = f[s][i] * raw_get(rx[s], i);
                        if (RST && (cuts >> s & 1)) hin[i] = u;                       // (w_ stands: nothing came through)
                        else { w_[s][i] = fmaf(-hin[i], rate[i] * sa[s][i], w_[s][i]); hin[i] = fmaf(a[s][i], hin[i], u); }
                    }
                xp += (S - 1) * k.d_sT; ap += (S - 1) * k.d_sT; ip += (S - 1) * k.d_sT;
#pragma unroll
                for (int s = S - 1; s >= 0; --s) {
                    const int t = t0 + s;
                    const bool live = t < Tb;
                    float ox[V], oa[V], oi[V];
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        const float gt = raw_get(rdy[s], i) + c[i], ag = a[s][i] * gt;
                        const float q = live ? ag * w_[s][i] : 0.f;
                        ox[i] = live ? gt * f[s][i] : 0.f;
                        oi[i] = ox[i] * xd[s][i];
                        oa[i] = fmaf(-q, sa[s][i], q);
                        dl[i] += q;
                        c[i] = RST && (cuts >> s & 1) ? 0.f : ag;
                    }
                    if (t < k.T) {
                        st_raw<T, V>(xp, raw_pack<T, V>(ox), nv);
                        st_raw<T, V>(ap, raw_pack<T, V>(oa), nv);
                        st_raw<T, V>(ip, raw_pack<T, V>(oi), nv);
                    }
                    xp -= k.d_sT; ap -= k.d_sT; ip -= k.d_sT;
                }
            } else {
                const float zero[V] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int s = 0; s < S; ++s) {
                    if (t0 + s < k.T) {
                        st_raw<T, V>(xp, raw_pack<T, V>(zero), nv);
                        st_raw<T, V>(ap, raw_pack<T, V>(zero), nv);
                        st_raw<T, V>(ip, raw_pack<T, V>(zero), nv);
                    }
                    xp += k.d_sT; ap += k.d_sT; ip += k.d_sT;
                }
            }
        }
        if (FINAL) load(tile - 1);
    }
    if (!FINAL) {
        if (wave == 0 && tw == 0) {
            const long o = ((long)b * k.nchunk + chunk) * k.C + c0;
#pragma unroll
            for (int i = 0; i < V; ++i)
                if (i < nv) { k.sumA[o + i] = ccut ? -1.f : cA[i]; k.sumH[o + i] = carry[i]; }
        }
        return;
    }
    if (k.dh0 && chunk == 0 && wave == 0 && tw == 0) {
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (i < nv) k.dh0[(long)b * k.C + c0 + i] = carry[i];
    }
    // the decay gradient's partial sum of this workgroup: time-threads, then waves, in a fixed order
#pragma unroll
    for (int i = 0; i < V; ++i)
#pragma unroll
        for (int d = TC; d < 64; d *= 2) dl[i] += __shfl_xor(dl[i], d);
    __syncthreads();
    if (tw == 0) {
#pragma unroll
        for (int i = 0; i < V; ++i) sA[0][wave][cl + i] = dl[i];
    }
    __syncthreads();
    const int e = threadIdx.x;
    if (e < CH && ch0 + e < k.C) k.part[((long)b * k.nchunk + chunk) * k.C + ch0 + e] = (sA[0][0][e] + sA[0][1][e]) + (sA[0][2][e] + sA[0][3][e]);
}

// One acting step: state rows are read, advanced and written back. Rows that name the same slot are consecutive steps of that state, in
// row order: the first of them does the work of all (a wave finds the others by comparing the slots, 64 at a time).
struct LinrecStepK {
    const void* x; const void* ga; const void* gi; long x_sB, ga_sB, gi_sB;
    const float* decay; float scale; const float* state; float* state_out; const int* slots;
    void* y; long y_sB; int B, C, D, n_slots;
};
template <class T>
__global__ void __launch_bounds__(64) linrec_step(const LinrecStepK k) {
    constexpr int VEC = VEC_OF<T>;
    const int row = blockIdx.x, lane = threadIdx.x;
    const int c0 = (int)(blockIdx.y * 64 + lane) * VEC, nv = min(max(k.C - c0, 0), VEC);
    T* y = (T*)k.y;
    int slot = row;
    if (k.slots) {
        slot = k.slots[row];
        if (slot < 0 || slot >= k.n_slots) {            // a padded row
            float z[VEC];
#pragma unroll
            for (int i = 0; i < VEC; ++i) z[i] = 0.f;
            st_raw<T>(y + (long)row * k.y_sB + c0, raw_pack<T>(z), nv);
            return;
        }
        for (int j = 0; j < row; j += 64)
            if (__any(j + lane < row && k.slots[j + lane] == slot)) return;
    }
    float rate[VEC], h[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
        rate[i] = i < nv ? k.scale * softplus_(k.decay[(c0 + i) % k.D]) : 0.f;
        h[i] = i < nv ? k.state[(long)slot * k.C + c0 + i] : 0.f;
    }
    int r = row;
    for (;;) {
        const auto rx = ld_raw<T>((const T*)k.x + (long)r * k.x_sB + c0, nv);
        const auto ra = ld_raw<T>((const T*)k.ga + (long)r * k.ga_sB + c0, nv);
        const auto ri = ld_raw<T>((const T*)k.gi + (long)r * k.gi_sB + c0, nv);
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            const LrGate g = lr_gate<true, false>(raw_get(ra, i), raw_get(ri, i), rate[i]);
            h[i] = fmaf(g.a, h[i], g.beta * (g.si * raw_get(rx, i)));
        }
        st_raw<T>(y + (long)r * k.y_sB + c0, raw_pack<T>(h), nv);
        if (!k.slots) break;
        int nxt = -1;
        for (int j = (r + 1) & ~63; j < k.B && nxt < 0; j += 64) {
            const unsigned long long m = __ballot(j + lane > r && j + lane < k.B && k.slots[j + lane < k.B ? j + lane : 0] == slot);
            if (m) nxt = j + __ffsll((long long)m) - 1;
        }
        if (nxt < 0) break;
        r = nxt;
    }
#pragma unroll
    for (int i = 0; i < VEC; ++i)
        if (i < nv) k.state_out[(long)slot * k.C + c0 + i] = h[i];
}

// ddecay[d] = sigmoid(decay) / softplus(decay) * sum_r part[r][d], rows in a fixed order: a wave's rows eight at a time, then the waves
__global__ void __launch_bounds__(1024) linrec_ddecay(const float* src, long R, int D, const float* decay, float* dst) {
    __shared__ float s[16][64];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, d = blockIdx.x * 64 + lane;
    float acc = 0.f;
    if (d < D) {
        long r = w;
        for (; r + 7 * 16 < R; r += 8 * 16) {
            float v[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = src[(r + j * 16) * D + d];
#pragma unroll
            for (int j = 0; j < 8; ++j) acc += v[j];
        }
        for (; r < R; r += 16) acc += src[r * D + d];
    }
    s[w][lane] = acc;
    __syncthreads();
    if (w == 0 && d < D) {
        float t = 0.f;
#pragma unroll
        for (int j = 0; j < 16; ++j) t += s[j][lane];
        const float v = decay[d], sp = softplus_(v);
        dst[d] = R ? t * (sp > 0.f ? (1.f / (1.f + expf(-v))) / sp : 1.f) : 0.f;        // (both vanish alike as decay -> -inf)
    }
}

struct LrPlan { int ncol, ntile, nchunk, tiles_per_chunk; };
static LrPlan lr_plan(const refil_linrec_desc& d, bool bwd) {
    LrPlan p;
    p.ncol = cdiv(d.C, lr_tc(d.dtype, d.B, d.C) * LR_V);
    p.ntile = cdiv(d.T, lr_tile(d.dtype, d.B, d.C));
    // Too few (episode, column) pairs to fill the card: the time axis is cut into chunks of whole tiles, at the price of reading the
    // inputs once more for the chunks' maps -- as many as the card holds at once (waves per SIMD by registers: launch bounds), so that
    // there is one round of workgroups and each starts once. (256 compute units of four SIMDs.)
    const bool wide = d.dtype == REFIL_F32;
    const long pairs = (long)d.B * p.ncol, hold = 256L * (bwd ? (wide ? 3 : 2) : (wide ? 4 : 3));
    long n = pairs > 0 ? hold / pairs : 1;
    if (n < 1) n = 1;
    if (n > p.ntile) n = p.ntile;
    if (n > 256) n = 256;
    p.tiles_per_chunk = n > 1 ? (int)cdivl(p.ntile, n) : p.ntile;
    p.nchunk = n > 1 ? cdiv(p.ntile, p.tiles_per_chunk) : 1;
    return p;
}
static int lr_check(const refil_linrec_desc& d, const char* who) {
    REFIL_CHECK(d.dtype >= REFIL_F32 && d.dtype <= REFIL_F16, "%s: dtype %d is none of REFIL_F32 / REFIL_BF16 / REFIL_F16", who, d.dtype);
    REFIL_CHECK(d.B >= 0 && d.T >= 0 && d.C >= 0 && d.D > 0, "%s: B %d, T %d, C %d must not be negative, D %d positive", who, d.B, d.T, d.C, d.D);
    REFIL_CHECK(d.C % d.D == 0, "%s: C %d must be a multiple of D %d", who, d.C, d.D);
    // (a launch holds fewer than 2^32 lanes)
    REFIL_CHECK((long)d.B * cdiv(d.C, 64) < (1L << 24) && d.T <= (1 << 30), "%s: B %d x C %d (64 channels a workgroup) or T %d too large", who, d.B, d.C, d.T);
    REFIL_CHECK(d.scale > 0.f && d.scale < 1e30f, "%s: scale must be positive and finite", who);
    return 0;
}
static LinrecK lr_args(const refil_linrec_desc& d, const LrPlan& p) {
    LinrecK k{};
    k.x = d.x; k.ga = d.ga; k.gi = d.gi; k.x_sB = d.x_sB; k.x_sT = d.x_sT; k.ga_sB = d.ga_sB; k.ga_sT = d.ga_sT; k.gi_sB = d.gi_sB; k.gi_sT = d.gi_sT;
    k.decay = d.decay; k.scale = d.scale; k.h0 = d.h0; k.reset = d.reset; k.rs_sB = d.rs_sB; k.rs_sT = d.rs_sT; k.lengths = d.lengths;
    k.y = d.y; k.y_sB = d.y_sB; k.y_sT = d.y_sT; k.h_last = d.h_last; k.saved = d.saved;
    k.dy = d.dy; k.dy_sB = d.dy_sB; k.dy_sT = d.dy_sT; k.dh_last = d.dh_last; k.dx = d.dx; k.dga = d.dga; k.dgi = d.dgi; k.d_sB = d.d_sB; k.d_sT = d.d_sT;
    k.dh0 = d.dh0;
    k.B = d.B; k.T = d.T; k.C = d.C; k.D = d.D; k.ch = lr_tc(d.dtype, d.B, d.C) * LR_V; k.ncol = p.ncol; k.nchunk = p.nchunk; k.tiles_per_chunk = p.tiles_per_chunk; k.ntile = p.ntile;
    return k;
}
// workspace: [sumA][sumH] (more than one chunk), backward: [part]
static long lr_sum_floats(const refil_linrec_desc& d, const LrPlan& p) { return p.nchunk > 1 ? 2L * d.B * p.nchunk * d.C : 0; }
static long lr_ws_floats(const refil_linrec_desc& d, const LrPlan& p, bool bwd) {
    long n = lr_sum_floats(d, p);
    if (bwd) {
        const long rows = (long)d.B * p.nchunk * (d.C / d.D);
        n += rows * d.D;
    }
    return n;
}

template <class T, bool FINAL>
static void lr_go_fwd(const LinrecK& k, dim3 grid, hipStream_t st) {
    if constexpr (sizeof(T) == 2) {
        if (k.ch == 256) {
            if (k.reset) hipLaunchKernelGGL((linrec_fwd<T, 64, FINAL, true>), grid, dim3(256), 0, st, k);
            else hipLaunchKernelGGL((linrec_fwd<T, 64, FINAL, false>), grid, dim3(256), 0, st, k);
            return;
        }
    }
    if (k.reset) hipLaunchKernelGGL((linrec_fwd<T, 16, FINAL, true>), grid, dim3(256), 0, st, k);
    else hipLaunchKernelGGL((linrec_fwd<T, 16, FINAL, false>), grid, dim3(256), 0, st, k);
}
template <class T, bool FINAL>
static void lr_go_bwd(const LinrecK& k, dim3 grid, hipStream_t st) {
    if constexpr (sizeof(T) == 2) {
        if (k.ch == 256) {
            if (k.reset) hipLaunchKernelGGL((linrec_bwd<T, 64, FINAL, true>), grid, dim3(256), 0, st, k);
            else hipLaunchKernelGGL((linrec_bwd<T, 64, FINAL, false>), grid, dim3(256), 0, st, k);
            return;
        }
    }
    if (k.reset) hipLaunchKernelGGL((linrec_bwd<T, 16, FINAL, true>), grid, dim3(256), 0, st, k);
    else hipLaunchKernelGGL((linrec_bwd<T, 16, FINAL, false>), grid, dim3(256), 0, st, k);
}
template <class T>
static int lr_forward(const refil_linrec_desc& d, hipStream_t st) {
    const LrPlan p = lr_plan(d, false);
    LinrecK k = lr_args(d, p);
    float* ws = (float*)d.workspace;
    k.sumA = ws; k.sumH = ws ? ws + (long)d.B * p.nchunk * d.C : nullptr;
    const dim3 grid(d.B * p.ncol, p.nchunk);
    const double n = (double)d.B * d.T * d.C;
    if (p.nchunk > 1) {
        ProfScope ps("linrec_fwd<summary>", 20 * n, 3 * n * sizeof(T), st);
        lr_go_fwd<T, false>(k, grid, st);
        REFIL_LAUNCH_CHECK();
    }
    ProfScope ps("linrec_fwd", 25 * n, 4 * n * sizeof(T), st);
    lr_go_fwd<T, true>(k, grid, st);
    REFIL_LAUNCH_CHECK();
    return 0;
}
static int lr_ddecay(const refil_linrec_desc& d, const float* part, long rows, hipStream_t st) {
    hipLaunchKernelGGL(linrec_ddecay, dim3(cdiv(d.D, 64)), dim3(1024), 0, st, part, rows, d.D, d.decay, d.ddecay);
    REFIL_LAUNCH_CHECK();
    return 0;
}
template <class T>
static int lr_backward(const refil_linrec_desc& d, hipStream_t st) {
    const LrPlan p = lr_plan(d, true);
    LinrecK k = lr_args(d, p);
    float* ws = (float*)d.workspace;
    k.sumA = ws; k.sumH = ws + (long)d.B * p.nchunk * d.C;
    k.part = ws + lr_sum_floats(d, p);
    const long rows = (long)d.B * p.nchunk * (d.C / d.D);
    const dim3 grid(d.B * p.ncol, p.nchunk);
    const double n = (double)d.B * d.T * d.C;
    if (p.nchunk > 1) {
        ProfScope ps("linrec_bwd<summary>", 20 * n, 2 * n * sizeof(T), st);
        lr_go_bwd<T, false>(k, grid, st);
        REFIL_LAUNCH_CHECK();
    }
    {
        ProfScope ps("linrec_bwd", 55 * n, 7 * n * sizeof(T), st);
        lr_go_bwd<T, true>(k, grid, st);
        REFIL_LAUNCH_CHECK();
    }
    return lr_ddecay(d, k.part, rows, st);
}
template <class T>
static int lr_step(const refil_linrec_step_desc& d, hipStream_t st) {
    LinrecStepK k{};
    k.x = d.x; k.ga = d.ga; k.gi = d.gi; k.x_sB = d.x_sB; k.ga_sB = d.ga_sB; k.gi_sB = d.gi_sB; k.decay = d.decay; k.scale = d.scale;
    k.state = d.state; k.state_out = d.state_out; k.slots = d.slots; k.y = d.y; k.y_sB = d.y_sB; k.B = d.B; k.C = d.C; k.D = d.D; k.n_slots = d.n_slots;
    const double n = (double)d.B * d.C;
    ProfScope ps("linrec_step", 25 * n, n * (4 * sizeof(T) + 8), st);
    hipLaunchKernelGGL((linrec_step<T>), dim3(d.B, cdiv(d.C, 64 * VEC_OF<T>)), dim3(64), 0, st, k);
    REFIL_LAUNCH_CHECK();
    return 0;
}

}  // namespace refil

using namespace refil;

extern "C" size_t refil_linrec_workspace_bytes(const refil_linrec_desc* d, int32_t backward) {
    if (!d || lr_check(*d, "refil_linrec_workspace_bytes")) return 0;
    return (size_t)lr_ws_floats(*d, lr_plan(*d, backward != 0), backward != 0) * sizeof(float);
}
extern "C" int64_t refil_linrec_saved_floats(const refil_linrec_desc* d) {
    if (!d || lr_check(*d, "refil_linrec_saved_floats")) return 0;
    return (int64_t)d->B * cdiv(d->T, lr_tile(d->dtype, d->B, d->C)) * d->C;
}
extern "C" int refil_linrec_forward(const refil_linrec_desc* d, void* stream) {
    REFIL_CHECK(d, "refil_linrec_forward: null desc");
    if (int rc = lr_check(*d, "refil_linrec_forward")) return rc;
    if (!d->B || !d->C) return 0;
    REFIL_CHECK(d->decay, "refil_linrec_forward: decay is NULL");
    REFIL_CHECK(!d->T || (d->x && d->ga && d->gi && d->y), "refil_linrec_forward: x, ga, gi and y are required");
    const size_t need = refil_linrec_workspace_bytes(d, 0);
    REFIL_CHECK(!need || (d->workspace && d->workspace_bytes >= need), "refil_linrec_forward: workspace of %zu bytes, %zu needed", d->workspace_bytes, need);
    hipStream_t st = (hipStream_t)stream;
    return d->dtype == REFIL_F32 ? lr_forward<float>(*d, st) : d->dtype == REFIL_BF16 ? lr_forward<bf16_t>(*d, st) : lr_forward<f16_t>(*d, st);
}
extern "C" int refil_linrec_backward(const refil_linrec_desc* d, void* stream) {
    REFIL_CHECK(d, "refil_linrec_backward: null desc");
    if (int rc = lr_check(*d, "refil_linrec_backward")) return rc;
    REFIL_CHECK(d->decay && d->ddecay, "refil_linrec_backward: decay and ddecay are required");
    REFIL_CHECK(!d->B || !d->C || !d->T || (d->x && d->ga && d->gi && d->dy && d->dx && d->dga && d->dgi && d->saved),
                "refil_linrec_backward: x, ga, gi, dy, dx, dga, dgi and saved are required");
    const size_t need = refil_linrec_workspace_bytes(d, 1);
    REFIL_CHECK(!need || (d->workspace && d->workspace_bytes >= need), "refil_linrec_backward: workspace of %zu bytes, %zu needed", d->workspace_bytes, need);
    hipStream_t st = (hipStream_t)stream;
    if (!d->B || !d->C) return lr_ddecay(*d, nullptr, 0, st);
    return d->dtype == REFIL_F32 ? lr_backward<float>(*d, st) : d->dtype == REFIL_BF16 ? lr_backward<bf16_t>(*d, st) : lr_backward<f16_t>(*d, st);
}
extern "C" int refil_linrec_step(const refil_linrec_step_desc* d, void* stream) {
    REFIL_CHECK(d, "refil_linrec_step: null desc");
    REFIL_CHECK(d->dtype >= REFIL_F32 && d->dtype <= REFIL_F16, "refil_linrec_step: dtype %d is none of REFIL_F32 / REFIL_BF16 / REFIL_F16", d->dtype);
    REFIL_CHECK(d->B >= 0 && d->C >= 0 && d->D > 0 && d->C % d->D == 0, "refil_linrec_step: B %d, C %d must not be negative, C a multiple of D %d", d->B, d->C, d->D);
    REFIL_CHECK(d->scale > 0.f && d->scale < 1e30f, "refil_linrec_step: scale must be positive and finite");
    REFIL_CHECK(d->slots || d->n_slots >= d->B, "refil_linrec_step: %d state rows for %d rows without slots", d->n_slots, d->B);
    REFIL_CHECK((long)d->C <= 65535L * 256 && (long)d->B < (1L << 26), "refil_linrec_step: B %d or C %d too large", d->B, d->C);
    if (!d->B || !d->C) return 0;
    REFIL_CHECK(d->x && d->ga && d->gi && d->decay && d->state && d->state_out && d->y, "refil_linrec_step: x, ga, gi, decay, state, state_out and y are required");
    hipStream_t st = (hipStream_t)stream;
    return d->dtype == REFIL_F32 ? lr_step<float>(*d, st) : d->dtype == REFIL_BF16 ? lr_step<bf16_t>(*d, st) : lr_step<f16_t>(*d, st);
}
