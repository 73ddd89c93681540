// Norms before and after a block, fused with the block's gate and residual scale (include/refil_hip.h: refil_norm_gate_*).
//
//   N(v; w) = v w / sqrt(mean(v^2) + eps)
//   y = alpha x + s sigmoid(g) N(o; w_post)          behind the block: its output o joins the residual stream x
//   n = N(y; w_pre)                                  in front of the next block
//
// One pass: a row lives in the registers of TPR threads (16 bytes of it each, K times), the two sums of squares are tree sums in fp32, and
// n is taken from the unrounded y. Backward, with e = dn w_pre, yh = y / rms(y), oh = o / rms(o):
//   d  = dy + (e - yh mean(e yh)) / rms(y),                     dx = alpha d
//   f  = d s sigmoid(g),  e2 = f w_post:                        do = (e2 - oh mean(e2 oh)) / rms(o)
//   dg = f oh w_post (1 - sigmoid(g)),  dw_post = sum f oh,  ds = sum d sigmoid(g) oh w_post,  dw_pre = sum dn yh
// y is computed again from x, o and g (no more bytes than reading it, and unrounded); mean(e yh) and the sum of y^2 share one reduction.
// The column sums stay in registers (the widest rows: in LDS) over a workgroup's rows, are joined in LDS, and a second launch adds the
// workgroups' partial rows in a fixed order: no atomics, the same result every time.
//
// Bound by memory: N 16384, D 2048 in bf16 with a gate takes 64 us forward (5 streams, 5.2 TB/s) and 102 us backward (8 streams, 5.3 TB/s; a
// large copy reaches 4.7 .. 4.9), N 41472, D 128 in fp32 with a fifth of its rows masked 17.5 + 29 us. Narrow rows share a workgroup so
// that a wave's loads stay whole lines; the next row's loads leave in front of this row's sums, which is what keeps memory busy through the
// barriers. Few rows (N 128, D 64: 3.7 us) are a launch and one round of latency.
#include "kernels.h"
#include "profile.h"
#include "vecio.h"

namespace refil {

struct NormGateK {
    const void* x; const void* o; const void* g; long x_s, o_s, g_s;
    const float* w_post; const float* scale; const float* w_pre; float alpha, eps;
    const uint8_t* mask;
    void* y; void* n; long y_s, n_s;
    const void* dy; const void* dn; long dy_s, dn_s;
    void* dx; void* d_o; void* dg; long dx_s, do_s, dg_s;
    float* part;                 // [3][blocks][D]: dw_post, ds, dw_pre
    long N; int D;
};

// Sums of NS values over the TPR threads of a row, in a fixed tree order: neighbours, quads, halves and rows of 16 lanes by DPP, the rest by
// shuffles, the waves of a wide row through LDS. The LDS slots alternate (`turn`), so one barrier per sum suffices; it orders LDS only and
// leaves the next row's loads in flight.
template <int CTRL> __device__ __forceinline__ float dpp_add(float v) {
    return v + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xF, 0xF, true));
}
template <int TPR, int NS>
__device__ __forceinline__ void row_sums(float (&v)[NS], float* s_red, int& turn) {
#pragma unroll
    for (int q = 0; q < NS; ++q) {
        v[q] = dpp_add<0xB1>(v[q]);             // lane ^ 1
        v[q] = dpp_add<0x4E>(v[q]);             // lane ^ 2
        v[q] = dpp_add<0x141>(v[q]);            // the other four of eight
        if constexpr (TPR >= 16) v[q] = dpp_add<0x140>(v[q]);      // the other eight of sixteen
        if constexpr (TPR >= 32) v[q] += __shfl_xor(v[q], 16);
        if constexpr (TPR >= 64) v[q] += __shfl_xor(v[q], 32);
    }
    if constexpr (TPR > 64) {
        constexpr int NW = TPR / 64;                       // waves of a row; the row groups of a workgroup are whole waves
        const int wave = threadIdx.x >> 6, g0 = wave / NW * NW;
        float* s = s_red + turn * 32;
        turn ^= 1;
        if ((threadIdx.x & 63) == 0) {
#pragma unroll
            for (int q = 0; q < NS; ++q) s[q * 16 + wave] = v[q];
        }
        lds_barrier();
#pragma unroll
        for (int q = 0; q < NS; ++q) {
            float t = 0.f;
#pragma unroll
            for (int i = 0; i < NW; ++i) t += s[q * 16 + g0 + i];
            v[q] = t;
        }
    }
}

// rows of 1024 threads: one workgroup fills a compute unit and its registers, so the column sums lie in LDS as far as it reaches (backward
// of N 8000, D 8192 in bf16 249 us = 4.2 TB/s, 417 with them in registers; N 2707, D 4505 in fp32 146 for 190)
template <class T> constexpr bool ng_col_lds(int tpr, int k, bool bwd) { return bwd && tpr == 1024 && 12 * tpr * k * VEC_OF<T> <= 128 * 1024; }

template <class T, int K>
struct NgRow { Raw<T> x[K], o[K], g[K]; };
template <class T, int K>
struct NgGrad { Raw<T> dy[K], dn[K]; };

// WEIGHTS: the weights stay in registers over the rows of the workgroup (else they are read again for every row: rows so wide that the
// registers do not reach). AHEAD: the next row's loads are issued in front of this row's sums.
template <class T, int TPR, int K, bool BWD, bool ENDS>
__global__ void __launch_bounds__(TPR > 256 ? TPR : 256) norm_gate_kernel(const NormGateK k) {
    constexpr int VEC = VEC_OF<T>, THREADS = TPR > 256 ? TPR : 256, GROUPS = THREADS / TPR;
    constexpr bool WEIGHTS = TPR < 1024, AHEAD = TPR < 1024;
    constexpr int KW = WEIGHTS ? K : 1;
    __shared__ float s_red[64];
    const int col = threadIdx.x % TPR, grp = threadIdx.x / TPR;
    const float inv_d = 1.f / (float)k.D;
    // the ragged end of a row is read as the row's last VEC elements, moved down by `back`: one load, where VEC single ones would keep the
    // wave waiting (rows of fewer than VEC elements do that, and the widest, whose registers are full). ENDS: compiled in; rows of 1024
    // threads have a kernel of their own for it (N 4000, D 5001 in bf16 148 us backward for 168, but D 8192 would pay 271 for 250)
    const bool ragged = ENDS && k.D % VEC != 0 && k.D >= VEC;
    int turn = 0, nv[K], back[K];
    float wp[KW][VEC], sc[KW][VEC], wq[KW][VEC];
    auto weights = [&](int j, float (&p)[VEC], float (&s)[VEC], float (&q)[VEC]) {
        const int c0 = (j * TPR + col) * VEC;
        auto get = [&](const float* w, float (&o)[VEC]) {
#pragma unroll
            for (int h = 0; h < VEC / 4; ++h) {
                const int n = min(max(nv[j] - h * 4, 0), 4);
                if (w) {
                    const auto r = ld_raw<float, 4>(w + c0 + h * 4, n);
#pragma unroll
                    for (int i = 0; i < 4; ++i) o[h * 4 + i] = raw_get(r, i);
                } else {
#pragma unroll
                    for (int i = 0; i < 4; ++i) o[h * 4 + i] = i < n ? 1.f : 0.f;
                }
            }
        };
        get(k.w_post, p);
        get(k.scale, s);
        get(k.w_pre, q);
    };
#pragma unroll
    for (int j = 0; j < K; ++j) {
        nv[j] = min(max(k.D - (j * TPR + col) * VEC, 0), VEC);
        back[j] = ragged && nv[j] > 0 ? VEC - nv[j] : 0;
        if constexpr (WEIGHTS) weights(j, wp[j], sc[j], wq[j]);
    }
    constexpr bool COL_LDS = ng_col_lds<T>(TPR, K, BWD);
    constexpr int KA = BWD && !COL_LDS ? K : 1;
    extern __shared__ __attribute__((aligned(16))) char ng_smem[];
    f32x4* const s_acc = reinterpret_cast<f32x4*>(ng_smem) + threadIdx.x;       // [3][K][VEC / 4][TPR], a thread's own columns
    float awp[KA][VEC], asc[KA][VEC], awq[KA][VEC];
    if (BWD) {
#pragma unroll
        for (int j = 0; j < KA; ++j)
#pragma unroll
            for (int i = 0; i < VEC; ++i) awp[j][i] = asc[j][i] = awq[j][i] = 0.f;
        if constexpr (COL_LDS) {
            for (int e = 0; e < 3 * K * VEC / 4; ++e) s_acc[e * TPR] = f32x4{0.f, 0.f, 0.f, 0.f};
        }
    }
    NgRow<T, K> a;
    NgGrad<T, BWD ? K : 1> b;
    // (every thread takes every round: the sums hold workgroup barriers)
    const long rounds = cdivl(k.N, (long)gridDim.x * GROUPS);
    auto row_of = [&](long it) { return (it * gridDim.x + blockIdx.x) * GROUPS + grp; };
    auto alive = [&](long r) { return r < k.N && !(k.mask && k.mask[r]); };
    auto load = [&](long r, bool live) {
#pragma unroll
        for (int j = 0; j < K; ++j) {
            const int c0 = (j * TPR + col) * VEC - back[j], n = live ? nv[j] + back[j] : 0;
            a.x[j] = ld_raw<T>((const T*)k.x + r * k.x_s + c0, n);
            a.o[j] = ld_raw<T>((const T*)k.o + r * k.o_s + c0, k.o ? n : 0);
            a.g[j] = ld_raw<T>((const T*)k.g + r * k.g_s + c0, k.g ? n : 0);
            if constexpr (BWD) {
                b.dy[j] = ld_raw<T>((const T*)k.dy + r * k.dy_s + c0, k.dy ? n : 0);
                b.dn[j] = ld_raw<T>((const T*)k.dn + r * k.dn_s + c0, k.dn ? n : 0);
            }
        }
    };
    bool live_next = alive(row_of(0));
    if (AHEAD) load(row_of(0), live_next);
    for (long it = 0; it < rounds; ++it) {
        const long r = row_of(it);
        const bool in = r < k.N, live = live_next;
        if (it + 1 < rounds) live_next = alive(row_of(it + 1));
        if (!AHEAD) load(r, live);
        NgRow<T, K> c = a;
        NgGrad<T, BWD ? K : 1> d = b;
        if (AHEAD && it + 1 < rounds) load(row_of(it + 1), live_next);
        if (ragged) {
#pragma unroll
            for (int j = 0; j < K; ++j) {
                c.x[j] = raw_down<T, VEC>(c.x[j], back[j]); c.o[j] = raw_down<T, VEC>(c.o[j], back[j]); c.g[j] = raw_down<T, VEC>(c.g[j], back[j]);
                if constexpr (BWD) { d.dy[j] = raw_down<T, VEC>(d.dy[j], back[j]); d.dn[j] = raw_down<T, VEC>(d.dn[j], back[j]); }
            }
        }
        float irms_o = 0.f;
        if (k.o) {
            float q[1] = {0.f};
#pragma unroll
            for (int j = 0; j < K; ++j)
#pragma unroll
                for (int i = 0; i < VEC; ++i) { const float v = raw_get(c.o[j], i); q[0] = fmaf(v, v, q[0]); }
            row_sums<TPR, 1>(q, s_red, turn);
            irms_o = __builtin_amdgcn_rsqf(fmaf(q[0], inv_d, k.eps));
        }
        float y[K][VEC], sg[K][VEC], q[2] = {0.f, 0.f};
#pragma unroll
        for (int j = 0; j < K; ++j) {
            if constexpr (!WEIGHTS) weights(j, wp[0], sc[0], wq[0]);
            const int w = WEIGHTS ? j : 0;
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                sg[j][i] = k.g ? fast_sigmoid(raw_get(c.g[j], i)) : 1.f;
                const float v = sc[w][i] * sg[j][i] * (raw_get(c.o[j], i) * irms_o * wp[w][i]);
                y[j][i] = fmaf(k.alpha, raw_get(c.x[j], i), v);
                q[0] = fmaf(y[j][i], y[j][i], q[0]);
                if constexpr (BWD) q[1] = fmaf(raw_get(d.dn[j], i) * wq[w][i], y[j][i], q[1]);
            }
        }
        float irms_y = 0.f;
        if constexpr (!BWD) {
            if (k.n) {
                float q1[1] = {q[0]};
                row_sums<TPR, 1>(q1, s_red, turn);
                irms_y = __builtin_amdgcn_rsqf(fmaf(q1[0], inv_d, k.eps));
            }
#pragma unroll
            for (int j = 0; j < K; ++j) {
                const int c0 = (j * TPR + col) * VEC, n = in ? nv[j] : 0, w = WEIGHTS ? j : 0;
                if (k.y) {
                    float v[VEC];
#pragma unroll
                    for (int i = 0; i < VEC; ++i) v[i] = live ? y[j][i] : 0.f;
                    st_raw<T, VEC>((T*)k.y + r * k.y_s + c0, raw_pack<T>(v), n);
                }
                if (k.n) {
                    if constexpr (!WEIGHTS) { if (K > 1) weights(j, wp[0], sc[0], wq[0]); }
                    float v[VEC];
#pragma unroll
                    for (int i = 0; i < VEC; ++i) v[i] = live ? y[j][i] * irms_y * wq[w][i] : 0.f;
                    st_raw<T, VEC>((T*)k.n + r * k.n_s + c0, raw_pack<T>(v), n);
                }
            }
        } else {
            float m = 0.f;
            if (k.dn) {
                row_sums<TPR, 2>(q, s_red, turn);
                irms_y = __builtin_amdgcn_rsqf(fmaf(q[0], inv_d, k.eps));
                m = q[1] * inv_d * irms_y;                                    // mean(e yh)
            }
            float e2o[1] = {0.f};
#pragma unroll
            for (int j = 0; j < K; ++j) {
                if constexpr (!WEIGHTS) { if (K > 1) weights(j, wp[0], sc[0], wq[0]); }
                const int w = WEIGHTS ? j : 0;
#pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    const float yh = y[j][i] * irms_y, dn = raw_get(d.dn[j], i);
                    const float dd = raw_get(d.dy[j], i) + irms_y * (dn * wq[w][i] - yh * m);
                    const float oh = raw_get(c.o[j], i) * irms_o, dg = dd * sg[j][i], f = dg * sc[w][i];
                    // (masked rows were read as zeros: they add zeros)
                    const int ja = COL_LDS ? 0 : j;
                    awq[ja][i] = fmaf(dn, yh, awq[ja][i]);
                    awp[ja][i] = fmaf(f, oh, awp[ja][i]);
                    asc[ja][i] = fmaf(dg, oh * wp[w][i], asc[ja][i]);
                    e2o[0] = fmaf(f * wp[w][i], oh, e2o[0]);
                    y[j][i] = dd;
                }
                if constexpr (COL_LDS) {
#pragma unroll
                    for (int h = 0; h < VEC / 4; ++h) {
                        f32x4* const at = s_acc + (j * (VEC / 4) + h) * TPR;
                        at[0] += f32x4{awp[0][4 * h], awp[0][4 * h + 1], awp[0][4 * h + 2], awp[0][4 * h + 3]};
                        at[K * VEC / 4 * TPR] += f32x4{asc[0][4 * h], asc[0][4 * h + 1], asc[0][4 * h + 2], asc[0][4 * h + 3]};
                        at[2 * K * VEC / 4 * TPR] += f32x4{awq[0][4 * h], awq[0][4 * h + 1], awq[0][4 * h + 2], awq[0][4 * h + 3]};
                    }
#pragma unroll
                    for (int i = 0; i < VEC; ++i) awp[0][i] = asc[0][i] = awq[0][i] = 0.f;
                }
            }
            float m2 = 0.f;
            if (k.o) { row_sums<TPR, 1>(e2o, s_red, turn); m2 = e2o[0] * inv_d; }
#pragma unroll
            for (int j = 0; j < K; ++j) {
                if constexpr (!WEIGHTS) { if (K > 1) weights(j, wp[0], sc[0], wq[0]); }
                const int c0 = (j * TPR + col) * VEC, n = in ? nv[j] : 0, w = WEIGHTS ? j : 0;
                float ox[VEC], oo[VEC], og[VEC];
#pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    const float dd = y[j][i], oh = raw_get(c.o[j], i) * irms_o, e2 = dd * sc[w][i] * sg[j][i] * wp[w][i];
                    ox[i] = k.alpha * dd;
                    oo[i] = irms_o * (e2 - oh * m2);
                    og[i] = e2 * oh * (1.f - sg[j][i]);
                }
                st_raw<T, VEC>((T*)k.dx + r * k.dx_s + c0, raw_pack<T>(ox), n);
                if (k.o) st_raw<T, VEC>((T*)k.d_o + r * k.do_s + c0, raw_pack<T>(oo), n);
                if (k.g) st_raw<T, VEC>((T*)k.dg + r * k.dg_s + c0, raw_pack<T>(og), n);
            }
        }
    }
    if constexpr (BWD) {
        // column sums of the workgroup: its row groups in order
        __shared__ float s_col[GROUPS > 1 ? THREADS * VEC : 1];
#pragma unroll
        for (int q = 0; q < 3; ++q) {
            float* dst = k.part + ((long)q * gridDim.x + blockIdx.x) * k.D;
#pragma unroll
            for (int j = 0; j < K; ++j) {
                const int c0 = (j * TPR + col) * VEC;
                if constexpr (COL_LDS) {
#pragma unroll
                    for (int h = 0; h < VEC / 4; ++h) {
                        const f32x4 t = s_acc[((q * K + j) * (VEC / 4) + h) * TPR];
                        const float v[4] = {t[0], t[1], t[2], t[3]};
                        st_raw<float, 4>(dst + c0 + h * 4, raw_pack<float, 4>(v), min(max(nv[j] - h * 4, 0), 4));
                    }
                    continue;
                }
                const int ja = COL_LDS ? 0 : j;
                const float (&acc)[VEC] = q == 0 ? awp[ja] : q == 1 ? asc[ja] : awq[ja];
                if constexpr (GROUPS == 1) {
#pragma unroll
                    for (int h = 0; h < VEC / 4; ++h) st_raw<float, 4>(dst + c0 + h * 4, raw_pack<float, 4>(acc + h * 4), min(max(nv[j] - h * 4, 0), 4));
                } else {
                    __syncthreads();
#pragma unroll
                    for (int i = 0; i < VEC; ++i) s_col[(grp * TPR + col) * VEC + i] = acc[i];
                    __syncthreads();
                    for (int c = threadIdx.x; c < TPR * VEC && c < k.D; c += THREADS) {
                        float t = 0.f;
#pragma unroll
                        for (int gi = 0; gi < GROUPS; ++gi) t += s_col[gi * TPR * VEC + c];
                        dst[c] = t;
                    }
                }
            }
        }
    }
}

// the three weight gradients: blockIdx.y picks the field; the partial rows are added in order, a wave's eight at a time
__global__ void __launch_bounds__(1024) norm_gate_colsum(const float* part, int R, int D, float* d0, float* d1, float* d2) {
    __shared__ float s[16][64];
    float* dst = blockIdx.y == 0 ? d0 : blockIdx.y == 1 ? d1 : d2;
    if (!dst) return;
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, d = blockIdx.x * 64 + lane;
    const float* src = part + (long)blockIdx.y * R * D;
    float acc = 0.f;
    if (d < D) {
        int r = w;
        for (; r + 7 * 16 < R; r += 8 * 16) {
            float v[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = src[(long)(r + j * 16) * D + d];
#pragma unroll
            for (int j = 0; j < 8; ++j) acc += v[j];
        }
        for (; r < R; r += 16) acc += src[(long)r * D + d];
    }
    s[w][lane] = acc;
    __syncthreads();
    if (w == 0 && d < D) {
        float t = 0.f;
#pragma unroll
        for (int j = 0; j < 16; ++j) t += s[j][lane];
        dst[d] = t;
    }
}

constexpr int NG_MAX_D = 16384;
constexpr int NG_BLOCKS = 512;       // workgroups of a backward launch at most (rows of 1024 threads: half): each leaves three partial rows of D sums

// (the threads of a row; of a row that ng_two halves, this many and half of them give the same launch)
static int ng_tpr(int D, int vec) {
    int t = 8;
    while (t < 1024 && t * vec < D) t *= 2;
    return t;
}
static int ng_groups(int tpr) { return tpr >= 256 ? 1 : 256 / tpr; }
// Rows of 513 .. 1024 vectors: 512 threads with two each, whose next row is in flight, against 1024 with one. N 3000, D 2500 in fp32 33 + 48 us
// against 45 + 59 (forward, backward); N 8000, D 5000 in bf16 120 against 131 forward, but backward the registers do not reach.
template <class T> constexpr bool ng_two(bool bwd) { return sizeof(T) == 4 || !bwd; }
static long ng_blocks(const refil_norm_gate_desc& d, bool bwd) {
    const int tpr = ng_tpr(d.D, d.dtype == REFIL_F32 ? 4 : 8);
    const long n = cdivl(d.N, ng_groups(tpr)), most = bwd ? (tpr == 1024 ? NG_BLOCKS / 2 : NG_BLOCKS) : 2048;
    return n < most ? n : most;
}

template <class T, int TPR, int K, bool ENDS>
static int ng_go(const NormGateK& k, bool bwd, long blocks, hipStream_t st) {
    const dim3 threads(TPR > 256 ? TPR : 256);
    // (rows of 513 .. 1024 vectors have one form in each direction: ng_two)
    if (!bwd) {
        if constexpr (TPR != 1024 || K > 1) hipLaunchKernelGGL((norm_gate_kernel<T, TPR, K, false, ENDS>), dim3(blocks), threads, 0, st, k);
    } else if constexpr (TPR != 512 || K == 1 || ng_two<T>(true)) {
        constexpr size_t LDS = ng_col_lds<T>(TPR, K, true) ? (size_t)12 * TPR * K * VEC_OF<T> : 0;
        if (LDS) REFIL_HIP(hipFuncSetAttribute((const void*)norm_gate_kernel<T, TPR, K, true, ENDS>, (hipFuncAttribute)hipFuncAttributeMaxDynamicSharedMemorySize, (int)LDS));
        hipLaunchKernelGGL((norm_gate_kernel<T, TPR, K, true, ENDS>), dim3(blocks), threads, LDS, st, k);
    }
    REFIL_LAUNCH_CHECK();
    return 0;
}
template <class T, int TPR, int K>
static int ng_run(const NormGateK& k, bool bwd, long blocks, hipStream_t st) {
    if constexpr (TPR == 1024) {
        if constexpr (K * VEC_OF<T> <= 8) { if (k.D % VEC_OF<T>) return ng_go<T, TPR, K, true>(k, bwd, blocks, st); }
        return ng_go<T, TPR, K, false>(k, bwd, blocks, st);
    } else return ng_go<T, TPR, K, true>(k, bwd, blocks, st);
}
template <class T>
static int ng_pick(const NormGateK& k, bool bwd, long blocks, hipStream_t st) {
    constexpr int VEC = VEC_OF<T>;
    static_assert(ng_two<T>(false), "the forward of 1024 vectors is the halved one");
    if (k.D > 512 * VEC && k.D <= 1024 * VEC && ng_two<T>(bwd)) return ng_run<T, 512, 2>(k, bwd, blocks, st);
    switch (ng_tpr(k.D, VEC)) {
        case 8: return ng_run<T, 8, 1>(k, bwd, blocks, st);
        case 16: return ng_run<T, 16, 1>(k, bwd, blocks, st);
        case 32: return ng_run<T, 32, 1>(k, bwd, blocks, st);
        case 64: return ng_run<T, 64, 1>(k, bwd, blocks, st);
        case 128: return ng_run<T, 128, 1>(k, bwd, blocks, st);
        case 256: return ng_run<T, 256, 1>(k, bwd, blocks, st);
        case 512: return ng_run<T, 512, 1>(k, bwd, blocks, st);
        default: break;
    }
    if constexpr (!ng_two<T>(true)) { if (k.D <= 1024 * VEC) return ng_run<T, 1024, 1>(k, bwd, blocks, st); }
    if (k.D <= 2048 * VEC) return ng_run<T, 1024, 2>(k, bwd, blocks, st);
    if constexpr (VEC == 4) return ng_run<T, 1024, 4>(k, bwd, blocks, st);
    set_error("refil_norm_gate: D %d too large", k.D);
    return 1;
}
static int ng_check(const refil_norm_gate_desc& d, const char* who) {
    REFIL_CHECK(d.dtype >= REFIL_F32 && d.dtype <= REFIL_F16, "%s: dtype %d is none of REFIL_F32 / REFIL_BF16 / REFIL_F16", who, d.dtype);
    REFIL_CHECK(d.N >= 0 && d.D > 0 && d.D <= NG_MAX_D, "%s: N %lld must not be negative, D %d in 1 .. %d", who, (long long)d.N, d.D, NG_MAX_D);
    REFIL_CHECK(d.eps >= 1.17549435e-38f && d.eps < 1e30f, "%s: eps must be positive (a normal fp32 number) and finite", who);
    REFIL_CHECK(!d.gate || d.o, "%s: a gate needs the block's output", who);
    return 0;
}
static NormGateK ng_args(const refil_norm_gate_desc& d) {
    NormGateK k{};
    k.x = d.x; k.o = d.o; k.g = d.gate; k.x_s = d.x_stride; k.o_s = d.o_stride; k.g_s = d.gate_stride;
    k.w_post = d.post_weight; k.scale = d.res_scale; k.w_pre = d.pre_weight; k.alpha = d.alpha; k.eps = d.eps; k.mask = d.row_mask;
    k.y = d.y; k.n = d.n; k.y_s = d.y_stride; k.n_s = d.n_stride;
    k.dy = d.dy; k.dn = d.dn; k.dy_s = d.dy_stride; k.dn_s = d.dn_stride;
    k.dx = d.dx; k.d_o = d.d_o; k.dg = d.dgate; k.dx_s = d.dx_stride; k.do_s = d.do_stride; k.dg_s = d.dgate_stride;
    k.N = d.N; k.D = d.D;
    return k;
}
static int ng_dispatch(const NormGateK& k, int dtype, bool bwd, long blocks, hipStream_t st) {
    const double n = (double)k.N * k.D, es = dtype == REFIL_F32 ? 4 : 2;
    const int has_o = k.o != nullptr, has_g = k.g != nullptr;
    const double streams = bwd ? 2 + 2 * has_o + 2 * has_g + (k.dy != nullptr) + (k.dn != nullptr) : 1 + has_o + has_g + (k.y != nullptr) + (k.n != nullptr);
    ProfScope ps(bwd ? "norm_gate_bwd" : "norm_gate_fwd", (bwd ? 50 : 20) * n, streams * n * es, st);
    return dtype == REFIL_F32 ? ng_pick<float>(k, bwd, blocks, st) : dtype == REFIL_BF16 ? ng_pick<bf16_t>(k, bwd, blocks, st) : ng_pick<f16_t>(k, bwd, blocks, st);
}

}  // namespace refil

using namespace refil;

extern "C" size_t refil_norm_gate_workspace_bytes(const refil_norm_gate_desc* d) {
    if (!d || ng_check(*d, "refil_norm_gate_workspace_bytes")) return 0;
    return (size_t)3 * ng_blocks(*d, true) * d->D * sizeof(float);
}
extern "C" int refil_norm_gate_forward(const refil_norm_gate_desc* d, void* stream) {
    REFIL_CHECK(d, "refil_norm_gate_forward: null desc");
    if (int rc = ng_check(*d, "refil_norm_gate_forward")) return rc;
    if (!d->N) return 0;
    REFIL_CHECK(d->y || d->n, "refil_norm_gate_forward: neither y nor n is asked for");
    REFIL_CHECK(d->x, "refil_norm_gate_forward: x is required");
    return ng_dispatch(ng_args(*d), d->dtype, false, ng_blocks(*d, false), (hipStream_t)stream);
}
extern "C" int refil_norm_gate_backward(const refil_norm_gate_desc* d, void* stream) {
    REFIL_CHECK(d, "refil_norm_gate_backward: null desc");
    if (int rc = ng_check(*d, "refil_norm_gate_backward")) return rc;
    REFIL_CHECK(!d->N || (d->x && (d->dy || d->dn) && d->dx), "refil_norm_gate_backward: x, dx and one of dy, dn are required");
    REFIL_CHECK(!d->N || !d->o || d->d_o, "refil_norm_gate_backward: d_o is required with o");
    REFIL_CHECK(!d->N || !d->gate || d->dgate, "refil_norm_gate_backward: dgate is required with gate");
    const size_t need = refil_norm_gate_workspace_bytes(d);
    REFIL_CHECK(!need || (d->workspace && d->workspace_bytes >= need), "refil_norm_gate_backward: workspace of %zu bytes, %zu needed", d->workspace_bytes, need);
    hipStream_t st = (hipStream_t)stream;
    NormGateK k = ng_args(*d);
    k.part = (float*)d->workspace;
    const long blocks = ng_blocks(*d, true);
    if (d->N)
        if (int rc = ng_dispatch(k, d->dtype, true, blocks, st)) return rc;
    if (d->dpost_weight || d->dres_scale || d->dpre_weight) {
        hipLaunchKernelGGL(norm_gate_colsum, dim3(cdiv(d->D, 64), 3), dim3(1024), 0, st, k.part, (int)blocks, d->D, d->dpost_weight, d->dres_scale, d->dpre_weight);
        REFIL_LAUNCH_CHECK();
    }
    return 0;
}
