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
// The column sums stay in registers over a workgroup's rows, are joined in LDS, and a second launch adds the workgroups' partial rows in
// a fixed order: no atomics, the same result every time.
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

template <int TPR>
__device__ __forceinline__ float row_sum(float v, float* s_red) {
    constexpr int W = TPR < 64 ? TPR : 64;
#pragma unroll
    for (int d = 1; d < W; d *= 2) v += __shfl_xor(v, d);
    if constexpr (TPR > 64) {
        constexpr int NW = TPR / 64;                       // waves of a row; the row groups of a workgroup are whole waves
        const int wave = threadIdx.x >> 6, g0 = wave / NW * NW;
        if ((threadIdx.x & 63) == 0) s_red[wave] = v;
        __syncthreads();
        float t = 0.f;
#pragma unroll
        for (int i = 0; i < NW; ++i) t += s_red[g0 + i];
        __syncthreads();
        v = t;
    }
    return v;
}

template <class T, int TPR, int K, bool BWD>
__global__ void __launch_bounds__(TPR > 256 ? TPR : 256) norm_gate_kernel(const NormGateK k) {
    constexpr int VEC = VEC_OF<T>, THREADS = TPR > 256 ? TPR : 256, GROUPS = THREADS / TPR;
    __shared__ float s_red[16];
    const int col = threadIdx.x % TPR, grp = threadIdx.x / TPR;
    const float inv_d = 1.f / (float)k.D;
    int nv[K];
    float wp[K][VEC], sc[K][VEC], wq[K][VEC];
#pragma unroll
    for (int j = 0; j < K; ++j) {
        const int c0 = (j * TPR + col) * VEC;
        nv[j] = min(max(k.D - c0, 0), VEC);
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            const bool in = i < nv[j];
            wp[j][i] = in ? (k.w_post ? k.w_post[c0 + i] : 1.f) : 0.f;
            sc[j][i] = in ? (k.scale ? k.scale[c0 + i] : 1.f) : 0.f;
            wq[j][i] = in ? (k.w_pre ? k.w_pre[c0 + i] : 1.f) : 0.f;
        }
    }
    float awp[BWD ? K : 1][VEC], asc[BWD ? K : 1][VEC], awq[BWD ? K : 1][VEC];
    if (BWD) {
#pragma unroll
        for (int j = 0; j < K; ++j)
#pragma unroll
            for (int i = 0; i < VEC; ++i) awp[j][i] = asc[j][i] = awq[j][i] = 0.f;
    }
    const long rounds = cdivl(k.N, (long)gridDim.x * GROUPS);
    for (long it = 0; it < rounds; ++it) {
        // (every thread takes every round: the reductions hold workgroup barriers)
        const long r = (it * gridDim.x + blockIdx.x) * GROUPS + grp;
        const bool in = r < k.N, live = in && !(k.mask && k.mask[r]);
        Raw<T> rx[K], ro[K], rg[K], rdy[K], rdn[K];
#pragma unroll
        for (int j = 0; j < K; ++j) {
            const int c0 = (j * TPR + col) * VEC, n = live ? nv[j] : 0;
            rx[j] = ld_raw<T>((const T*)k.x + r * k.x_s + c0, n);
            ro[j] = ld_raw<T>((const T*)k.o + r * k.o_s + c0, k.o ? n : 0);
            rg[j] = ld_raw<T>((const T*)k.g + r * k.g_s + c0, k.g ? n : 0);
            if (BWD) {
                rdy[j] = ld_raw<T>((const T*)k.dy + r * k.dy_s + c0, k.dy ? n : 0);
                rdn[j] = ld_raw<T>((const T*)k.dn + r * k.dn_s + c0, k.dn ? n : 0);
            }
        }
        float irms_o = 0.f;
        if (k.o) {
            float q = 0.f;
#pragma unroll
            for (int j = 0; j < K; ++j)
#pragma unroll
                for (int i = 0; i < VEC; ++i) { const float v = raw_get(ro[j], i); q = fmaf(v, v, q); }
            irms_o = __builtin_amdgcn_rsqf(fmaf(row_sum<TPR>(q, s_red), inv_d, k.eps));
        }
        float y[K][VEC], sg[K][VEC], q = 0.f, ey = 0.f;
#pragma unroll
        for (int j = 0; j < K; ++j)
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                sg[j][i] = k.g ? fast_sigmoid(raw_get(rg[j], i)) : 1.f;
                const float v = sc[j][i] * sg[j][i] * (raw_get(ro[j], i) * irms_o * wp[j][i]);
                y[j][i] = fmaf(k.alpha, raw_get(rx[j], i), v);
                q = fmaf(y[j][i], y[j][i], q);
                if (BWD) ey = fmaf(raw_get(rdn[j], i) * wq[j][i], y[j][i], ey);
            }
        float irms_y = 0.f;
        if (BWD ? k.dn != nullptr : k.n != nullptr) irms_y = __builtin_amdgcn_rsqf(fmaf(row_sum<TPR>(q, s_red), inv_d, k.eps));
        if (!BWD) {
#pragma unroll
            for (int j = 0; j < K; ++j) {
                const int c0 = (j * TPR + col) * VEC, n = in ? nv[j] : 0;
                if (k.y) {
                    float v[VEC];
#pragma unroll
                    for (int i = 0; i < VEC; ++i) v[i] = live ? y[j][i] : 0.f;
                    st_raw<T>((T*)k.y + r * k.y_s + c0, raw_pack<T>(v), n);
                }
                if (k.n) {
                    float v[VEC];
#pragma unroll
                    for (int i = 0; i < VEC; ++i) v[i] = live ? y[j][i] * irms_y * wq[j][i] : 0.f;
                    st_raw<T>((T*)k.n + r * k.n_s + c0, raw_pack<T>(v), n);
                }
            }
        } else {
            float m = 0.f;
            if (k.dn) m = row_sum<TPR>(ey, s_red) * inv_d * irms_y;          // mean(e yh)
            float e2o = 0.f;
#pragma unroll
            for (int j = 0; j < K; ++j)
#pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    const float yh = y[j][i] * irms_y, dn = raw_get(rdn[j], i);
                    const float d = raw_get(rdy[j], i) + irms_y * (dn * wq[j][i] - yh * m);
                    awq[j][i] = live ? fmaf(dn, yh, awq[j][i]) : awq[j][i];
                    const float oh = raw_get(ro[j], i) * irms_o, f = d * sc[j][i] * sg[j][i];
                    awp[j][i] = live ? fmaf(f, oh, awp[j][i]) : awp[j][i];
                    asc[j][i] = live ? fmaf(d * sg[j][i], oh * wp[j][i], asc[j][i]) : asc[j][i];
                    e2o = fmaf(f * wp[j][i], oh, e2o);
                    y[j][i] = d;
                }
            float m2 = 0.f;
            if (k.o) m2 = row_sum<TPR>(e2o, s_red) * inv_d;
#pragma unroll
            for (int j = 0; j < K; ++j) {
                const int c0 = (j * TPR + col) * VEC, n = in ? nv[j] : 0;
                float ox[VEC], oo[VEC], og[VEC];
#pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    const float d = y[j][i], oh = raw_get(ro[j], i) * irms_o, f = d * sc[j][i] * sg[j][i];
                    ox[i] = live ? k.alpha * d : 0.f;
                    oo[i] = live ? irms_o * (f * wp[j][i] - oh * m2) : 0.f;
                    og[i] = live ? f * oh * wp[j][i] * (1.f - sg[j][i]) : 0.f;
                }
                st_raw<T>((T*)k.dx + r * k.dx_s + c0, raw_pack<T>(ox), n);
                if (k.o) st_raw<T>((T*)k.d_o + r * k.do_s + c0, raw_pack<T>(oo), n);
                if (k.g) st_raw<T>((T*)k.dg + r * k.dg_s + c0, raw_pack<T>(og), n);
            }
        }
    }
    if (BWD) {
        // column sums of the workgroup: its row groups in order
        __shared__ float s_col[GROUPS > 1 ? THREADS * VEC : 1];
#pragma unroll
        for (int q = 0; q < 3; ++q) {
            float* dst = k.part + ((long)q * gridDim.x + blockIdx.x) * k.D;
#pragma unroll
            for (int j = 0; j < K; ++j) {
                const int c0 = (j * TPR + col) * VEC;
                const float (&acc)[VEC] = q == 0 ? awp[j] : q == 1 ? asc[j] : awq[j];
                if constexpr (GROUPS == 1) {
#pragma unroll
                    for (int i = 0; i < VEC; ++i)
                        if (i < nv[j]) dst[c0 + i] = acc[i];
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

// the three weight gradients: blockIdx.y picks the field, the partial rows are added in order
__global__ void __launch_bounds__(1024) norm_gate_colsum(const float* part, int R, int D, float* d0, float* d1, float* d2) {
    __shared__ float s[16][64];
    float* dst = blockIdx.y == 0 ? d0 : blockIdx.y == 1 ? d1 : d2;
    if (!dst) return;
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, d = blockIdx.x * 64 + lane;
    const float* src = part + (long)blockIdx.y * R * D;
    float acc = 0.f;
    if (d < D)
        for (int r = w; r < R; r += 16) acc += src[(long)r * D + d];
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
constexpr int NG_BLOCKS = 512;       // workgroups of a backward launch at most: each leaves three partial rows of D sums

static int ng_tpr(int D, int vec) {
    int t = 8;
    while (t < 1024 && t * vec < D) t *= 2;
    return t;
}
static int ng_groups(int tpr) { return tpr >= 256 ? 1 : 256 / tpr; }
static long ng_blocks(const refil_norm_gate_desc& d, bool bwd) {
    const int tpr = ng_tpr(d.D, d.dtype == REFIL_F32 ? 4 : 8);
    const long n = cdivl(d.N, ng_groups(tpr)), most = bwd ? NG_BLOCKS : 4096;
    return n < most ? n : most;
}

template <class T, int TPR, int K>
static int ng_run(const NormGateK& k, bool bwd, long blocks, hipStream_t st) {
    if (bwd) hipLaunchKernelGGL((norm_gate_kernel<T, TPR, K, true>), dim3(blocks), dim3(TPR > 256 ? TPR : 256), 0, st, k);
    else hipLaunchKernelGGL((norm_gate_kernel<T, TPR, K, false>), dim3(blocks), dim3(TPR > 256 ? TPR : 256), 0, st, k);
    REFIL_LAUNCH_CHECK();
    return 0;
}
template <class T>
static int ng_pick(const NormGateK& k, bool bwd, long blocks, hipStream_t st) {
    constexpr int VEC = VEC_OF<T>;
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
    if (k.D <= 1024 * VEC) return ng_run<T, 1024, 1>(k, bwd, blocks, st);
    if (k.D <= 2048 * VEC) return ng_run<T, 1024, 2>(k, bwd, blocks, st);
    if constexpr (VEC == 4) return ng_run<T, 1024, 4>(k, bwd, blocks, st);
    set_error("refil_norm_gate: D %d too large", k.D);
    return 1;
}
static int ng_check(const refil_norm_gate_desc& d, const char* who) {
    REFIL_CHECK(d.dtype >= REFIL_F32 && d.dtype <= REFIL_F16, "%s: dtype %d is none of REFIL_F32 / REFIL_BF16 / REFIL_F16", who, d.dtype);
    REFIL_CHECK(d.N >= 0 && d.D > 0 && d.D <= NG_MAX_D, "%s: N %lld must not be negative, D %d in 1 .. %d", who, (long long)d.N, d.D, NG_MAX_D);
    REFIL_CHECK(d.eps > 0.f, "%s: eps must be positive", who);
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
