// Gated linear recurrence over an episode, forward / backward / one acting step (include/refil_hip.h: refil_linrec_*).
//
//   L_t = c softplus(decay) sigmoid(ga_t),  a_t = exp(-L_t)
//   h_t = [no reset at t] a_t h_{t-1} + sqrt(1 - a_t^2) sigmoid(gi_t) x_t,   y_t = h_t
//
// The gates do not read h, so a step is the affine map h -> A h + H and maps compose: (A2, H2) o (A1, H1) = (A2 A1, A2 H1 + H2). Time is
// cut three times: a thread composes S consecutive steps, a wave its 64 / TC time-threads by shuffles, a workgroup its four waves through
// LDS; the carry goes from 64-step tile to tile in registers. A reset cuts the chain: it travels beside the map as a flag instead of as
// A = 0, so that a NaN or Inf in front of it does not pass (0 * NaN).
//
// Backward: with g_t the whole gradient of h_t, g_t = dy_t + c_t and c_{t-1} = a_t g_t [no reset at t] -- the same maps A in reverse
// order, R_t in H_t's place. h_{t-1} is computed again from the fp32 state that the forward keeps at every tile's start (one value per
// 64 steps), not read from the rounded y: no 16-bit rounding enters the gradient, and 7 streams move where reading y would make 8.
// The gate gradients come without a division by sqrt(1 - a^2):
//   q_t = d loss / d log L_t = g_t (sigmoid(gi) x a^2 L / sqrt(1 - a^2) - a h_{t-1} L),   L / sqrt(1 - a^2) -> sqrt(L / 2) -> 0
//   dga_t = q_t (1 - sigmoid(ga)),   ddecay = sum q_t sigmoid(decay) / softplus(decay)
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
    int B, T, C, D, ncol, nchunk, tiles_per_chunk, ntile;
    float* sumA; float* sumH;          // [B][nchunk][C]: the maps of whole chunks (A = -1: the chunk holds a reset)
};

constexpr int LR_CH = 64;              // channels of a workgroup
constexpr int LR_TT = 64;              // steps of a tile = 4 waves x TW time-threads x S steps
constexpr int LR_WAVES = 4;

template <class T> struct LrGeo {
    static constexpr int VEC = VEC_OF<T>, TC = LR_CH / VEC, TW = 64 / TC, S = LR_TT / (LR_WAVES * TW);
};

// 1 - exp(-z), z >= 0, given e = exp(-z): the difference loses digits below z = 1/4, the series does not (next term z^8 / 40320)
__device__ __forceinline__ float one_minus_exp(float z, float e) {
    float p = fmaf(z, 1.98412698e-4f, -1.38888889e-3f);
    p = fmaf(z, p, 8.33333333e-3f);
    p = fmaf(z, p, -4.16666667e-2f);
    p = fmaf(z, p, 1.66666667e-1f);
    p = fmaf(z, p, -0.5f);
    p = fmaf(z, p, 1.0f);
    return z < 0.25f ? z * p : 1.0f - e;
}
__device__ __forceinline__ float softplus_(float v) { return fmaxf(v, 0.f) + log1pf(expf(-fabsf(v))); }

struct LrGate { float sa, si, L, a, beta, lob; };      // lob = L / sqrt(1 - a^2)
template <class T>
__device__ __forceinline__ LrGate lr_gate(float ga, float gi, float rate) {
    LrGate g;
    g.sa = sigmoid_t<T>(ga); g.si = sigmoid_t<T>(gi);
    g.L = rate * g.sa;
    g.a = exp_t<T>(-g.L);
    const float om = one_minus_exp(2.f * g.L, g.a * g.a);
    const float rs = __builtin_amdgcn_rsqf(fmaxf(om, 1e-37f));
    g.beta = om * rs;
    g.lob = g.L * rs;
    return g;
}

// rates of the workgroup's 64 channels, one softplus each
__device__ __forceinline__ void lr_rates(const LinrecK& k, int ch0, float* s_rate) {
    if (threadIdx.x < LR_CH) {
        const int c = ch0 + (int)threadIdx.x;
        s_rate[threadIdx.x] = c < k.C ? k.scale * softplus_(k.decay[c % k.D]) : 0.f;
    }
    __syncthreads();
}

// BWD = false: the maps' H from x; true: R from dy. One workgroup per (episode, 64 channels, chunk): the chunk's whole map.
// FINAL: also write the outputs, starting from the carry of the chunks in front (behind).
template <class T, bool FINAL>
__global__ void __launch_bounds__(256) linrec_fwd(const LinrecK k) {
    using G = LrGeo<T>;
    constexpr int VEC = G::VEC, TC = G::TC, TW = G::TW, S = G::S;
    __shared__ float s_rate[LR_CH];
    __shared__ float sA[2][LR_WAVES][LR_CH], sH[2][LR_WAVES][LR_CH];
    __shared__ int sCut[2][LR_WAVES];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int b = (int)(blockIdx.x / k.ncol), ch0 = (int)(blockIdx.x % k.ncol) * LR_CH, chunk = blockIdx.y;
    const int cl = (lane % TC) * VEC, c0 = ch0 + cl, nv = min(max(k.C - c0, 0), VEC);
    const int tw = lane / TC;
    lr_rates(k, ch0, s_rate);
    float rate[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) rate[i] = s_rate[cl + i];
    const int Tb = k.lengths ? min(max(k.lengths[b], 0), k.T) : k.T;
    float carry[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) carry[i] = FINAL && k.h0 && i < nv ? k.h0[(long)b * k.C + c0 + i] : 0.f;
    if (FINAL) {
        for (int j = 0; j < chunk; ++j) {
            const long o = ((long)b * k.nchunk + j) * k.C + c0;
#pragma unroll
            for (int i = 0; i < VEC; ++i)
                if (i < nv) { const float A = k.sumA[o + i], H = k.sumH[o + i]; carry[i] = A < 0.f ? H : fmaf(A, carry[i], H); }
        }
    }
    float cA[VEC]; int ccut = 0;       // !FINAL: the chunk's map so far (its H is `carry`, started from zero)
#pragma unroll
    for (int i = 0; i < VEC; ++i) cA[i] = 1.f;
    const T* xb = (const T*)k.x + (long)b * k.x_sB + c0;
    const T* gab = (const T*)k.ga + (long)b * k.ga_sB + c0;
    const T* gib = (const T*)k.gi + (long)b * k.gi_sB + c0;
    const int tile0 = chunk * k.tiles_per_chunk, tile1 = min(tile0 + k.tiles_per_chunk, k.ntile);
    for (int tile = tile0; tile < tile1; ++tile) {
        const int p = tile & 1, t0 = tile * LR_TT + (wave * TW + tw) * S;
        float a[S][VEC], u[S][VEC], A[VEC], H[VEC];
        bool cut[S]; int anycut = 0;
        Raw rx[S], rga[S], rgi[S];
#pragma unroll
        for (int s = 0; s < S; ++s) {
            const long t = t0 + s;
            const int n = t < Tb ? nv : 0;
            rx[s] = ld_raw<T>(xb + t * k.x_sT, n); rga[s] = ld_raw<T>(gab + t * k.ga_sT, n); rgi[s] = ld_raw<T>(gib + t * k.gi_sT, n);
            cut[s] = k.reset && t < Tb && k.reset[(long)b * k.rs_sB + t * k.rs_sT] != 0;
            anycut |= (int)cut[s];
        }
#pragma unroll
        for (int i = 0; i < VEC; ++i) { A[i] = 1.f; H[i] = 0.f; }
#pragma unroll
        for (int s = 0; s < S; ++s) {
            const bool live = t0 + s < Tb;
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                const LrGate g = lr_gate<T>(raw_get<T>(rga[s], i), raw_get<T>(rgi[s], i), rate[i]);
                a[s][i] = live ? g.a : 1.f;                       // past the end the state stays as it is
                u[s][i] = live ? g.beta * g.si * raw_get<T>(rx[s], i) : 0.f;
                H[i] = cut[s] ? u[s][i] : fmaf(a[s][i], H[i], u[s][i]);
                A[i] *= a[s][i];
            }
        }
        // inclusive over the wave's time-threads, then exclusive
#pragma unroll
        for (int d = 1; d < TW; d *= 2) {
            const int pc = __shfl_up(anycut, d * TC);
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                const float pA = __shfl_up(A[i], d * TC), pH = __shfl_up(H[i], d * TC);
                if (tw >= d) { H[i] = anycut ? H[i] : fmaf(A[i], pH, H[i]); A[i] *= pA; }
            }
            if (tw >= d) anycut |= pc;
        }
        if (tw == TW - 1) {
#pragma unroll
            for (int i = 0; i < VEC; ++i) { sA[p][wave][cl + i] = A[i]; sH[p][wave][cl + i] = H[i]; }
            if (lane % TC == 0) sCut[p][wave] = anycut;
        }
        float eA[VEC], eH[VEC]; int ecut = __shfl_up(anycut, TC);
#pragma unroll
        for (int i = 0; i < VEC; ++i) { eA[i] = __shfl_up(A[i], TC); eH[i] = __shfl_up(H[i], TC); }
        if (tw == 0) {
            ecut = 0;
#pragma unroll
            for (int i = 0; i < VEC; ++i) { eA[i] = 1.f; eH[i] = 0.f; }
        }
        lds_barrier();
        float h[VEC];
        if (FINAL && k.saved && wave == 0 && tw == 0) {
            float* o = k.saved + ((long)b * k.ntile + tile) * k.C + c0;
#pragma unroll
            for (int i = 0; i < VEC; ++i)
                if (i < nv) o[i] = carry[i];
        }
#pragma unroll
        for (int w = 0; w < LR_WAVES; ++w) {
            const int wc = sCut[p][w];
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                if (w == wave) h[i] = carry[i];
                const float wA = sA[p][w][cl + i], wH = sH[p][w][cl + i];
                carry[i] = wc ? wH : fmaf(wA, carry[i], wH);
                if (!FINAL) cA[i] *= wA;
            }
            ccut |= wc;
        }
        if (FINAL) {
#pragma unroll
            for (int i = 0; i < VEC; ++i) h[i] = ecut ? eH[i] : fmaf(eA[i], h[i], eH[i]);
#pragma unroll
            for (int s = 0; s < S; ++s) {
                const long t = t0 + s;
                float o[VEC];
#pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    h[i] = cut[s] ? u[s][i] : fmaf(a[s][i], h[i], u[s][i]);
                    o[i] = t < Tb ? h[i] : 0.f;
                }
                if (t < k.T) st_raw<T>((T*)k.y + (long)b * k.y_sB + t * k.y_sT + c0, raw_pack<T>(o), nv);
            }
        }
    }
    if (wave == 0 && tw == 0) {
        if (!FINAL) {
            const long o = ((long)b * k.nchunk + chunk) * k.C + c0;
#pragma unroll
            for (int i = 0; i < VEC; ++i)
                if (i < nv) { k.sumA[o + i] = ccut ? -1.f : cA[i]; k.sumH[o + i] = carry[i]; }
        } else if (k.h_last && chunk == k.nchunk - 1) {
#pragma unroll
            for (int i = 0; i < VEC; ++i)
                if (i < nv) k.h_last[(long)b * k.C + c0 + i] = carry[i];
        }
    }
}

template <class T, bool FINAL>
__global__ void __launch_bounds__(256) linrec_bwd(const LinrecK k) {
    using G = LrGeo<T>;
    constexpr int VEC = G::VEC, TC = G::TC, TW = G::TW, S = G::S;
    __shared__ float s_rate[LR_CH];
    __shared__ float sA[2][LR_WAVES][LR_CH], sH[2][LR_WAVES][LR_CH], sR[2][LR_WAVES][LR_CH];
    __shared__ int sCut[2][LR_WAVES];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int b = (int)(blockIdx.x / k.ncol), ch0 = (int)(blockIdx.x % k.ncol) * LR_CH, chunk = blockIdx.y;
    const int cl = (lane % TC) * VEC, c0 = ch0 + cl, nv = min(max(k.C - c0, 0), VEC);
    const int tw = lane / TC;
    lr_rates(k, ch0, s_rate);
    float rate[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) rate[i] = s_rate[cl + i];
    const int Tb = k.lengths ? min(max(k.lengths[b], 0), k.T) : k.T;
    float carry[VEC], cA[VEC], dl[VEC]; int ccut = 0;
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
        carry[i] = FINAL && k.dh_last && i < nv ? k.dh_last[(long)b * k.C + c0 + i] : 0.f;
        cA[i] = 1.f; dl[i] = 0.f;
    }
    if (FINAL) {
        for (int j = k.nchunk - 1; j > chunk; --j) {
            const long o = ((long)b * k.nchunk + j) * k.C + c0;
#pragma unroll
            for (int i = 0; i < VEC; ++i)
                if (i < nv) { const float A = k.sumA[o + i], R = k.sumH[o + i]; carry[i] = A < 0.f ? R : fmaf(A, carry[i], R); }
        }
    }
    const T* xb = (const T*)k.x + (long)b * k.x_sB + c0;
    const T* gab = (const T*)k.ga + (long)b * k.ga_sB + c0;
    const T* gib = (const T*)k.gi + (long)b * k.gi_sB + c0;
    const T* dyb = (const T*)k.dy + (long)b * k.dy_sB + c0;
    const int tile0 = chunk * k.tiles_per_chunk, tile1 = min(tile0 + k.tiles_per_chunk, k.ntile);
    for (int tile = tile1 - 1; tile >= tile0; --tile) {
        const int p = tile & 1, t0 = tile * LR_TT + (wave * TW + tw) * S;
        Raw rx[S], rga[S], rgi[S], rdy[S];
        bool cut[S]; int anycut = 0;
#pragma unroll
        for (int s = 0; s < S; ++s) {
            const long t = t0 + s;
            const int n = t < Tb ? nv : 0;
            rga[s] = ld_raw<T>(gab + t * k.ga_sT, n); rdy[s] = ld_raw<T>(dyb + t * k.dy_sT, n);
            if (FINAL) { rx[s] = ld_raw<T>(xb + t * k.x_sT, n); rgi[s] = ld_raw<T>(gib + t * k.gi_sT, n); }
            cut[s] = k.reset && t < Tb && k.reset[(long)b * k.rs_sB + t * k.rs_sT] != 0;
            anycut |= (int)cut[s];
        }
        float hin[VEC];
        if (FINAL) {
            const float* o = k.saved + ((long)b * k.ntile + tile) * k.C + c0;
#pragma unroll
            for (int i = 0; i < VEC; ++i) hin[i] = i < nv ? o[i] : 0.f;
        }
        LrGate g[S][VEC];
        float A[VEC], H[VEC], R[VEC];
#pragma unroll
        for (int i = 0; i < VEC; ++i) { A[i] = 1.f; H[i] = 0.f; R[i] = 0.f; }
#pragma unroll
        for (int s = 0; s < S; ++s) {
            const bool live = t0 + s < Tb;
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                g[s][i] = lr_gate<T>(raw_get<T>(rga[s], i), FINAL ? raw_get<T>(rgi[s], i) : 0.f, rate[i]);
                if (!live) { g[s][i].a = 1.f; g[s][i].beta = 0.f; }
                if (FINAL) {
                    const float u = g[s][i].beta * g[s][i].si * raw_get<T>(rx[s], i);
                    H[i] = cut[s] ? u : fmaf(g[s][i].a, H[i], u);
                }
                A[i] *= g[s][i].a;
            }
        }
#pragma unroll
        for (int s = S - 1; s >= 0; --s)
#pragma unroll
            for (int i = 0; i < VEC; ++i) R[i] = cut[s] ? 0.f : g[s][i].a * (raw_get<T>(rdy[s], i) + R[i]);
        // forward: inclusive prefix of (A, H); backward: inclusive suffix of (B, R)
        float Bq[VEC]; int fcut = anycut, rcut = anycut;
#pragma unroll
        for (int i = 0; i < VEC; ++i) Bq[i] = A[i];
#pragma unroll
        for (int d = 1; d < TW; d *= 2) {
            const int pc = __shfl_up(fcut, d * TC), nc = __shfl_down(rcut, d * TC);
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                if (FINAL) {
                    const float pA = __shfl_up(A[i], d * TC), pH = __shfl_up(H[i], d * TC);
                    if (tw >= d) { H[i] = fcut ? H[i] : fmaf(A[i], pH, H[i]); A[i] *= pA; }
                }
                const float nA = __shfl_down(Bq[i], d * TC), nR = __shfl_down(R[i], d * TC);
                if (tw + d < TW) { R[i] = rcut ? R[i] : fmaf(Bq[i], nR, R[i]); Bq[i] *= nA; }
            }
            if (tw >= d) fcut |= pc;
            if (tw + d < TW) rcut |= nc;
        }
        if (tw == 0) {
#pragma unroll
            for (int i = 0; i < VEC; ++i) { sA[p][wave][cl + i] = Bq[i]; sR[p][wave][cl + i] = R[i]; }
            if (lane % TC == 0) sCut[p][wave] = rcut;
        }
        if (FINAL && tw == TW - 1) {
#pragma unroll
            for (int i = 0; i < VEC; ++i) sH[p][wave][cl + i] = H[i];
        }
        float eA[VEC], eH[VEC], xA[VEC], xR[VEC]; int ecut, xcut;
        if (FINAL) {
            ecut = __shfl_up(fcut, TC); xcut = __shfl_down(rcut, TC);
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                eA[i] = __shfl_up(A[i], TC); eH[i] = __shfl_up(H[i], TC);
                xA[i] = __shfl_down(Bq[i], TC); xR[i] = __shfl_down(R[i], TC);
            }
            if (tw == 0) {
                ecut = 0;
#pragma unroll
                for (int i = 0; i < VEC; ++i) { eA[i] = 1.f; eH[i] = 0.f; }
            }
            if (tw == TW - 1) {
                xcut = 0;
#pragma unroll
                for (int i = 0; i < VEC; ++i) { xA[i] = 1.f; xR[i] = 0.f; }
            }
        }
        lds_barrier();
        float c[VEC];
#pragma unroll
        for (int w = LR_WAVES - 1; w >= 0; --w) {
            const int wc = sCut[p][w];
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                if (w == wave) c[i] = carry[i];
                const float wA = sA[p][w][cl + i], wR = sR[p][w][cl + i];
                carry[i] = wc ? wR : fmaf(wA, carry[i], wR);
                if (!FINAL) cA[i] *= wA;
            }
            ccut |= wc;
        }
        if (FINAL) {
#pragma unroll
            for (int w = 0; w < LR_WAVES - 1; ++w) {
                if (w < wave) {
                    const int wc = sCut[p][w];
#pragma unroll
                    for (int i = 0; i < VEC; ++i) hin[i] = wc ? sH[p][w][cl + i] : fmaf(sA[p][w][cl + i], hin[i], sH[p][w][cl + i]);
                }
            }
            float hp[S][VEC];
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                hin[i] = ecut ? eH[i] : fmaf(eA[i], hin[i], eH[i]);
                c[i] = xcut ? xR[i] : fmaf(xA[i], c[i], xR[i]);
            }
#pragma unroll
            for (int s = 0; s < S; ++s)
#pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    hp[s][i] = hin[i];
                    const float u = g[s][i].beta * g[s][i].si * raw_get<T>(rx[s], i);
                    hin[i] = cut[s] ? u : fmaf(g[s][i].a, hin[i], u);
                }
#pragma unroll
            for (int s = S - 1; s >= 0; --s) {
                const long t = t0 + s;
                const bool live = t < Tb;
                float ox[VEC], oa[VEC], oi[VEC];
#pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    const LrGate& e = g[s][i];
                    const float gt = raw_get<T>(rdy[s], i) + c[i];
                    const float sx = e.si * raw_get<T>(rx[s], i);
                    const float through = cut[s] ? 0.f : e.a * hp[s][i] * e.L;
                    const float q = gt * (sx * e.a * e.a * e.lob - through);
                    ox[i] = live ? gt * e.beta * e.si : 0.f;
                    oi[i] = live ? gt * e.beta * sx * (1.f - e.si) : 0.f;
                    oa[i] = live ? q * (1.f - e.sa) : 0.f;
                    dl[i] += live ? q : 0.f;
                    c[i] = cut[s] ? 0.f : e.a * gt;
                }
                if (t < k.T) {
                    const long o = (long)b * k.d_sB + t * k.d_sT + c0;
                    st_raw<T>((T*)k.dx + o, raw_pack<T>(ox), nv);
                    st_raw<T>((T*)k.dga + o, raw_pack<T>(oa), nv);
                    st_raw<T>((T*)k.dgi + o, raw_pack<T>(oi), nv);
                }
            }
        }
    }
    if (!FINAL) {
        if (wave == 0 && tw == 0) {
            const long o = ((long)b * k.nchunk + chunk) * k.C + c0;
#pragma unroll
            for (int i = 0; i < VEC; ++i)
                if (i < nv) { k.sumA[o + i] = ccut ? -1.f : cA[i]; k.sumH[o + i] = carry[i]; }
        }
        return;
    }
    if (k.dh0 && chunk == 0 && wave == 0 && tw == 0) {
#pragma unroll
        for (int i = 0; i < VEC; ++i)
            if (i < nv) k.dh0[(long)b * k.C + c0 + i] = carry[i];
    }
    // the decay gradient's partial sum of this workgroup: time-threads, then waves, in a fixed order
#pragma unroll
    for (int i = 0; i < VEC; ++i)
#pragma unroll
        for (int d = TC; d < 64; d *= 2) dl[i] += __shfl_xor(dl[i], d);
    __syncthreads();
    if (tw == 0) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) sA[0][wave][cl + i] = dl[i];
    }
    __syncthreads();
    if (wave == 0 && ch0 + lane < k.C)
        k.part[((long)b * k.nchunk + chunk) * k.C + ch0 + lane] = (sA[0][0][lane] + sA[0][1][lane]) + (sA[0][2][lane] + sA[0][3][lane]);
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
        const Raw rx = ld_raw<T>((const T*)k.x + (long)r * k.x_sB + c0, nv);
        const Raw ra = ld_raw<T>((const T*)k.ga + (long)r * k.ga_sB + c0, nv);
        const Raw ri = ld_raw<T>((const T*)k.gi + (long)r * k.gi_sB + c0, nv);
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            const LrGate g = lr_gate<T>(raw_get<T>(ra, i), raw_get<T>(ri, i), rate[i]);
            h[i] = fmaf(g.a, h[i], g.beta * g.si * raw_get<T>(rx, i));
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

// out[d] = factor(d) * sum_r src[r][d], rows in a fixed order. decay != NULL: factor = sigmoid(decay) / softplus(decay).
__global__ void __launch_bounds__(256) colsum_stage(const float* src, long R, int D, long rows_per, float* dst) {
    __shared__ float s[4][64];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, d = blockIdx.x * 64 + lane;
    const long r0 = (long)blockIdx.y * rows_per, r1 = min(r0 + rows_per, R);
    float acc = 0.f;
    if (d < D)
        for (long r = r0 + w; r < r1; r += 4) acc += src[r * D + d];
    s[w][lane] = acc;
    __syncthreads();
    if (w == 0 && d < D) dst[(long)blockIdx.y * D + d] = (s[0][lane] + s[1][lane]) + (s[2][lane] + s[3][lane]);
}
__global__ void __launch_bounds__(1024) colsum_final(const float* src, long R, int D, const float* decay, float* dst) {
    __shared__ float s[16][64];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, d = blockIdx.x * 64 + lane;
    float acc = 0.f;
    if (d < D)
        for (long r = w; r < R; r += 16) acc += src[r * D + d];
    s[w][lane] = acc;
    __syncthreads();
    if (w == 0 && d < D) {
        float t = 0.f;
#pragma unroll
        for (int j = 0; j < 16; ++j) t += s[j][lane];
        if (decay) {
            const float v = decay[d], sp = softplus_(v);
            t *= sp > 0.f ? (1.f / (1.f + expf(-v))) / sp : 1.f;        // (both vanish alike as decay -> -inf)
        }
        dst[d] = t;
    }
}
long colsum_tmp_floats(long R, int D) { return R > 512 ? 256L * D : 0; }
int colsum_launch(const float* src, long R, int D, float* tmp, const float* decay, float* dst, hipStream_t st) {
    const dim3 cols(cdiv(D, 64));
    if (R > 512) {
        const long per = cdivl(R, 256);
        const int n = (int)cdivl(R, per);
        hipLaunchKernelGGL(colsum_stage, dim3(cdiv(D, 64), n), dim3(256), 0, st, src, R, D, per, tmp);
        REFIL_LAUNCH_CHECK();
        src = tmp; R = n;
    }
    hipLaunchKernelGGL(colsum_final, cols, dim3(1024), 0, st, src, R, D, decay, dst);
    REFIL_LAUNCH_CHECK();
    return 0;
}

struct LrPlan { int ncol, ntile, nchunk, tiles_per_chunk; };
static LrPlan lr_plan(const refil_linrec_desc& d) {
    LrPlan p;
    p.ncol = cdiv(d.C, LR_CH);
    p.ntile = cdiv(d.T, LR_TT);
    p.nchunk = 1;
    p.tiles_per_chunk = p.ntile;
    return p;
}
static int lr_check(const refil_linrec_desc& d, const char* who) {
    REFIL_CHECK(d.dtype >= REFIL_F32 && d.dtype <= REFIL_F16, "%s: dtype %d is none of REFIL_F32 / REFIL_BF16 / REFIL_F16", who, d.dtype);
    REFIL_CHECK(d.B >= 0 && d.T >= 0 && d.C >= 0 && d.D > 0, "%s: B %d, T %d, C %d must not be negative, D %d positive", who, d.B, d.T, d.C, d.D);
    REFIL_CHECK(d.C % d.D == 0, "%s: C %d must be a multiple of D %d", who, d.C, d.D);
    REFIL_CHECK((long)d.B * cdiv(d.C, LR_CH) < (1L << 31) && d.T <= (1 << 30), "%s: B %d x C %d x T %d too large", who, d.B, d.C, d.T);
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
    k.B = d.B; k.T = d.T; k.C = d.C; k.D = d.D; k.ncol = p.ncol; k.nchunk = p.nchunk; k.tiles_per_chunk = p.tiles_per_chunk; k.ntile = p.ntile;
    return k;
}
// workspace: [sumA][sumH] (more than one chunk), backward: [part][column-sum scratch]
static long lr_sum_floats(const refil_linrec_desc& d, const LrPlan& p) { return p.nchunk > 1 ? 2L * d.B * p.nchunk * d.C : 0; }
static long lr_ws_floats(const refil_linrec_desc& d, const LrPlan& p, bool bwd) {
    long n = lr_sum_floats(d, p);
    if (bwd) {
        const long rows = (long)d.B * p.nchunk * (d.C / d.D);
        n += rows * d.D + colsum_tmp_floats(rows, d.D);
    }
    return n;
}

template <class T>
static int lr_forward(const refil_linrec_desc& d, hipStream_t st) {
    const LrPlan p = lr_plan(d);
    LinrecK k = lr_args(d, p);
    float* ws = (float*)d.workspace;
    k.sumA = ws; k.sumH = ws ? ws + (long)d.B * p.nchunk * d.C : nullptr;
    const dim3 grid(d.B * p.ncol, p.nchunk);
    const double n = (double)d.B * d.T * d.C;
    if (p.nchunk > 1) {
        ProfScope ps("linrec_fwd<summary>", 20 * n, 3 * n * sizeof(T), st);
        hipLaunchKernelGGL((linrec_fwd<T, false>), grid, dim3(256), 0, st, k);
        REFIL_LAUNCH_CHECK();
    }
    ProfScope ps("linrec_fwd", 25 * n, 4 * n * sizeof(T), st);
    hipLaunchKernelGGL((linrec_fwd<T, true>), grid, dim3(256), 0, st, k);
    REFIL_LAUNCH_CHECK();
    return 0;
}
template <class T>
static int lr_backward(const refil_linrec_desc& d, hipStream_t st) {
    const LrPlan p = lr_plan(d);
    LinrecK k = lr_args(d, p);
    float* ws = (float*)d.workspace;
    k.sumA = ws; k.sumH = ws + (long)d.B * p.nchunk * d.C;
    k.part = ws + lr_sum_floats(d, p);
    const long rows = (long)d.B * p.nchunk * (d.C / d.D);
    const dim3 grid(d.B * p.ncol, p.nchunk);
    const double n = (double)d.B * d.T * d.C;
    if (p.nchunk > 1) {
        ProfScope ps("linrec_bwd<summary>", 20 * n, 2 * n * sizeof(T), st);
        hipLaunchKernelGGL((linrec_bwd<T, false>), grid, dim3(256), 0, st, k);
        REFIL_LAUNCH_CHECK();
    }
    {
        ProfScope ps("linrec_bwd", 55 * n, 7 * n * sizeof(T), st);
        hipLaunchKernelGGL((linrec_bwd<T, true>), grid, dim3(256), 0, st, k);
        REFIL_LAUNCH_CHECK();
    }
    return colsum_launch(k.part, rows, d.D, k.part + rows * d.D, d.decay, d.ddecay, st);
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
    return (size_t)lr_ws_floats(*d, lr_plan(*d), backward != 0) * sizeof(float);
}
extern "C" int64_t refil_linrec_saved_floats(const refil_linrec_desc* d) {
    if (!d || lr_check(*d, "refil_linrec_saved_floats")) return 0;
    return (int64_t)d->B * cdiv(d->T, LR_TT) * d->C;
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
    if (!d->B || !d->C) return colsum_launch(nullptr, 0, d->D, nullptr, nullptr, d->ddecay, st);
    return d->dtype == REFIL_F32 ? lr_backward<float>(*d, st) : d->dtype == REFIL_BF16 ? lr_backward<bf16_t>(*d, st) : lr_backward<f16_t>(*d, st);
}
extern "C" int refil_linrec_step(const refil_linrec_step_desc* d, void* stream) {
    REFIL_CHECK(d, "refil_linrec_step: null desc");
    REFIL_CHECK(d->dtype >= REFIL_F32 && d->dtype <= REFIL_F16, "refil_linrec_step: dtype %d is none of REFIL_F32 / REFIL_BF16 / REFIL_F16", d->dtype);
    REFIL_CHECK(d->B >= 0 && d->C >= 0 && d->D > 0 && d->C % d->D == 0, "refil_linrec_step: B %d, C %d must not be negative, C a multiple of D %d", d->B, d->C, d->D);
    REFIL_CHECK(d->scale > 0.f && d->scale < 1e30f, "refil_linrec_step: scale must be positive and finite");
    REFIL_CHECK(d->slots || d->n_slots >= d->B, "refil_linrec_step: %d state rows for %d rows without slots", d->n_slots, d->B);
    REFIL_CHECK((long)d->C <= 65535L * 256, "refil_linrec_step: C %d too large", d->C);
    if (!d->B || !d->C) return 0;
    REFIL_CHECK(d->x && d->ga && d->gi && d->decay && d->state && d->state_out && d->y, "refil_linrec_step: x, ga, gi, decay, state, state_out and y are required");
    hipStream_t st = (hipStream_t)stream;
    return d->dtype == REFIL_F32 ? lr_step<float>(*d, st) : d->dtype == REFIL_BF16 ? lr_step<bf16_t>(*d, st) : lr_step<f16_t>(*d, st);
}
