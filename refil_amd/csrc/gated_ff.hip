// Gated feed-forward block h = act(x Wg^T + bg) * (x Wu^T + bu), forward and backward (include/refil_hip.h: refil_gated_ff_*).
//
// All products are C[m][n] = sum_k A[m][k] B[n][k] with both operands k-contiguous in 16 bits, on v_mfma_f32_16x16x32 (fp32 accumulate):
//   forward   A = x, B = [Wg | Wu] interleaved so that one wave holds both projections of a column: bias, activation and product happen
//             in its registers; h (and for training the two pre-activations) is all that is written
//   backward  [dg | du] from the saved pre-activations and dh (one elementwise pass that also leaves the transposed copy and the bias
//             sums); dx = [dg | du] [Wg ; Wu] with the weights transposed once per call; [dWg ; dWu] = [dg | du]^T x
// fp32 operands are split exactly into three bf16 pieces and a product runs as six bf16 products (hi hi, hi mid, mid hi, mid mid, hi lo,
// lo hi), as the library's projection GEMMs do: the k loop walks the six pairs of planes.
// Up to 64 rows the weights' bytes are the cost and a second kernel reads them once, straight into matrix-core fragments.
#include "kernels.h"
#include "profile.h"
#include "split.h"
#include "vecio.h"

namespace refil {

typedef __bf16 gf_bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 gf_f16x8 __attribute__((ext_vector_type(8)));
typedef unsigned gf_u32x4 __attribute__((ext_vector_type(4)));

template <class E>
__device__ __forceinline__ f32x4 gf_mfma(gf_u32x4 a, gf_u32x4 b, f32x4 c) {
    if constexpr (__is_same(E, f16_t)) return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(gf_f16x8, a), __builtin_bit_cast(gf_f16x8, b), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(gf_bf16x8, a), __builtin_bit_cast(gf_bf16x8, b), c, 0, 0, 0);
}

// the six products of two three-way splits that reach 2^-24 of the result, leading one last (smallest terms first)
__host__ __device__ constexpr int gf_pair_a(int p) { return p == 0 ? 2 : p == 1 ? 0 : p == 2 ? 1 : p == 3 ? 1 : p == 4 ? 0 : 0; }
__host__ __device__ constexpr int gf_pair_b(int p) { return p == 0 ? 0 : p == 1 ? 2 : p == 2 ? 1 : p == 3 ? 0 : p == 4 ? 1 : 0; }

// ---- activation ----
// gelu(v) = v/2 (1 + tanh(A (v + B v^3)))
constexpr float GF_A = 0.797884560802865f, GF_B = 0.044715f;
__device__ __forceinline__ float gf_act(int act, float v) {
    if (act == REFIL_ACT_SILU) return v * fast_sigmoid(v);
    // 1 + tanh(z) = 2 sigmoid(2 z): no cancellation on the negative side
    return v * fast_sigmoid(2.f * GF_A * (v + GF_B * v * v * v));
}
// value and derivative
__device__ __forceinline__ void gf_act_grad(int act, float v, float& f, float& df) {
    if (act == REFIL_ACT_SILU) {
        const float s = fast_sigmoid(v);
        f = v * s;
        df = s * (1.f + v * (1.f - s));
    } else {
        const float s = fast_sigmoid(2.f * GF_A * (v + GF_B * v * v * v));
        f = v * s;
        df = s + v * s * (1.f - s) * (2.f * GF_A) * (1.f + 3.f * GF_B * v * v);
    }
}

// ---- the tiled product ----
struct GfGemm {
    const void* A; long lda, planeA;
    const void* B0; const void* B1; long ldb, planeB;        // B1: the second half of the interleaved forward
    int M, N, K, pairs;                                      // K a multiple of 64, zero-padded
    int splits; float* partial;                              // splits > 1: fp32 partial sums [splits][M][N]
    void* C0; void* C1; long ldc; int msplit;                // rows >= msplit go to C1 (dWg / dWu)
    // gated epilogue
    const void* bias0; const void* bias1; void* save0; void* save1; int act;
};

constexpr int GF_BK = 64;

__device__ __forceinline__ void gf_copy16(const void* g, void* lds) {
    // 64 lanes x 16 bytes of global memory to 1 KB of LDS behind `lds` (wave-uniform), lane order
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)g, (__attribute__((address_space(3))) void*)lds, 16, 0, 0);
}

// WM x WN waves, each MT x NT tiles of 16 x 16. LDS rows hold 64 k values = 8 chunks of 16 bytes, chunk c of row r in slot c ^ (r & 7):
// the fragment reads (16 rows, one chunk) hit all banks, and the swizzle costs nothing on the way in (it permutes the lanes' addresses).
template <class T, class E, int WM, int WN, int MT, int NT, bool GATED>
__global__ void __launch_bounds__(WM * WN * 64) gf_gemm(const GfGemm k) {
    constexpr int WAVES = WM * WN, BM = WM * MT * 16, BN = WN * NT * 16, HALF = GATED ? BN / 2 : BN;
    constexpr int A_IT = BM / 8 / WAVES, B_IT = BN / 8 / WAVES;
    extern __shared__ __attribute__((aligned(16))) char gf_smem[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int wm = wave / WN, wn = wave % WN;
    const int mt = cdiv(k.M, BM), nt = cdiv(k.N, HALF);
    // consecutive workgroups land on different XCDs (8 of them): give each XCD a contiguous run of tiles, in 8-row panels, so that its
    // L2 holds the panels it reads
    const int total = mt * nt;
    int id = blockIdx.x;
    {
        const int per = total / 8, rem = total % 8, xcd = id % 8, pos = id / 8;
        id = xcd * per + min(xcd, rem) + pos;
    }
    const int panel = id / (8 * nt), prow = min(8, mt - panel * 8), in_panel = id - panel * 8 * nt;
    const int m0 = (panel * 8 + in_panel % prow) * BM, n0 = in_panel / prow * HALF;
    const int split = blockIdx.y;

    const E* pa[A_IT]; const E* pb[B_IT];
#pragma unroll
    for (int i = 0; i < A_IT; ++i) {
        const int r = (i * WAVES + wave) * 8 + (lane >> 3), ch = (lane & 7) ^ (r & 7);
        pa[i] = (const E*)k.A + (long)min(m0 + r, k.M - 1) * k.lda + ch * 8;
    }
#pragma unroll
    for (int i = 0; i < B_IT; ++i) {
        const int r = (i * WAVES + wave) * 8 + (lane >> 3), ch = (lane & 7) ^ (r & 7);
        const E* src = (const E*)k.B0;
        int n = n0 + r;
        if (GATED) {      // rows of a wave's columns: NT/2 tiles of the gate, then the same columns of the up projection
            const int w = r / (NT * 16), j = r % (NT * 16);
            if (j >= NT * 8) src = (const E*)k.B1;
            n = n0 + w * NT * 8 + j % (NT * 8);
        }
        pb[i] = src + (long)min(n, k.N - 1) * k.ldb + ch * 8;
    }
    const int kb = k.K / GF_BK, iters = kb * k.pairs;
    const int per = cdiv(iters, k.splits), it0 = min(split * per, iters), it1 = min(it0 + per, iters);
    char* const sa = gf_smem; char* const sb = gf_smem + 2 * BM * 128;

    auto stage = [&](int it, int buf) {
        const int p = it / kb, kk = it - p * kb;
        const long oa = (k.pairs > 1 ? gf_pair_a(p) * k.planeA : 0) + (long)kk * GF_BK, ob = (k.pairs > 1 ? gf_pair_b(p) * k.planeB : 0) + (long)kk * GF_BK;
#pragma unroll
        for (int i = 0; i < A_IT; ++i) gf_copy16(pa[i] + oa, sa + buf * BM * 128 + (i * WAVES + wave) * 1024);
#pragma unroll
        for (int i = 0; i < B_IT; ++i) gf_copy16(pb[i] + ob, sb + buf * BN * 128 + (i * WAVES + wave) * 1024);
    };

    f32x4 acc[MT][NT];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

    if (it0 < it1) stage(it0, 0);
    __syncthreads();
    for (int it = it0; it < it1; ++it) {
        const int buf = (it - it0) & 1;
        if (it + 1 < it1) stage(it + 1, buf ^ 1);
        const char* a = sa + buf * BM * 128 + wm * MT * 16 * 128;
        const char* b = sb + buf * BN * 128 + wn * NT * 16 * 128;
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
            const int r = lane & 15, slot = ((kk * 4 + (lane >> 4)) ^ (r & 7)) * 16;
            gf_u32x4 fa[MT], fb[NT];
#pragma unroll
            for (int i = 0; i < MT; ++i) fa[i] = *reinterpret_cast<const gf_u32x4*>(a + (i * 16 + r) * 128 + slot);
#pragma unroll
            for (int j = 0; j < NT; ++j) fb[j] = *reinterpret_cast<const gf_u32x4*>(b + (j * 16 + r) * 128 + slot);
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int j = 0; j < NT; ++j) acc[i][j] = gf_mfma<E>(fb[j], fa[i], acc[i][j]);      // D rows = n, columns = m: a lane holds 4 neighbouring n
        }
        __syncthreads();
    }

    // lane: m = lane & 15, n = 4 (lane >> 4) + 0..3 of every tile
#pragma unroll
    for (int i = 0; i < MT; ++i) {
        const int m = m0 + (wm * MT + i) * 16 + (lane & 15);
        if (m >= k.M) continue;
        if constexpr (GATED) {
#pragma unroll
            for (int j = 0; j < NT / 2; ++j) {
                const int n = n0 + wn * NT * 8 + j * 16 + (lane >> 4) * 4;
                float g[4], u[4], h[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    g[r] = acc[i][j][r]; u[r] = acc[i][j + NT / 2][r];
                    if (k.bias0 && n + r < k.N) g[r] += to_f32(((const T*)k.bias0)[n + r]);
                    if (k.bias1 && n + r < k.N) u[r] += to_f32(((const T*)k.bias1)[n + r]);
                    h[r] = gf_act(k.act, g[r]) * u[r];
                }
                T* c = (T*)k.C0 + (long)m * k.ldc + n;
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (n + r < k.N) c[r] = from_f32<T>(h[r]);
                if (k.save0) {
                    T* s0 = (T*)k.save0 + (long)m * k.N + n; T* s1 = (T*)k.save1 + (long)m * k.N + n;
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (n + r < k.N) { s0[r] = from_f32<T>(g[r]); s1[r] = from_f32<T>(u[r]); }
                }
            }
        } else {
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                const int n = n0 + (wn * NT + j) * 16 + (lane >> 4) * 4;
                if (k.splits > 1) {
                    float* c = k.partial + ((long)split * k.M + m) * k.N + n;
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (n + r < k.N) c[r] = acc[i][j][r];
                } else {
                    T* c = (m < k.msplit ? (T*)k.C0 + (long)m * k.ldc : (T*)k.C1 + (long)(m - k.msplit) * k.ldc) + n;
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (n + r < k.N) c[r] = from_f32<T>(acc[i][j][r]);
                }
            }
        }
    }
}

// sums of the split products, in split order
template <class T>
__global__ void __launch_bounds__(256) gf_reduce(const float* partial, int splits, int M, int N, void* C0, void* C1, long ldc, int msplit) {
    const long n = (long)M * N;
    for (long e = (long)blockIdx.x * 256 + threadIdx.x; e < n; e += (long)gridDim.x * 256) {
        float s = 0.f;
        for (int p = 0; p < splits; ++p) s += partial[p * n + e];
        const int m = (int)(e / N), c = (int)(e - (long)m * N);
        T* o = m < msplit ? (T*)C0 + (long)m * ldc : (T*)C1 + (long)(m - msplit) * ldc;
        o[c] = from_f32<T>(s);
    }
}

// ---- operands into k-contiguous, zero-padded 16-bit form ----
template <class T> struct GfElem { typedef T type; static constexpr int planes = 1; };
template <> struct GfElem<float> { typedef bf16_t type; static constexpr int planes = 3; };

template <class T>
__device__ __forceinline__ void gf_emit(void* dst, long plane, long o, float v) {
    typedef typename GfElem<T>::type E;
    E* d = (E*)dst;
    if constexpr (GfElem<T>::planes == 1) d[o] = from_f32<T>(v);
    else {
        const E h = (E)v; const float r1 = v - (float)h;
        const E m = (E)r1; const float r2 = r1 - (float)m;
        d[o] = h; d[o + plane] = m; d[o + 2 * plane] = (E)r2;
    }
}
// dst[r][c] = src[r][c], c in [0, Kp)
template <class T>
__global__ void __launch_bounds__(256) gf_pack(const void* src, long ld, long rows, int K, int Kp, void* dst, long ldd, long plane) {
    const long n = rows * Kp;
    for (long e = (long)blockIdx.x * 256 + threadIdx.x; e < n; e += (long)gridDim.x * 256) {
        const long r = e / Kp; const int c = (int)(e - r * Kp);
        gf_emit<T>(dst, plane, r * ldd + c, c < K ? to_f32(((const T*)src)[r * ld + c]) : 0.f);
    }
}
// dst[c][r] = src[r][c], r in [0, Rp): 64 x 64 tiles through LDS
template <class T>
__global__ void __launch_bounds__(256) gf_transpose(const void* src, long ld, long rows, int cols, long Rp, void* dst, long ldd, long plane) {
    __shared__ float t[64][65];
    const long r0 = (long)blockIdx.x * 64; const int c0 = blockIdx.y * 64, l = threadIdx.x & 63, q = threadIdx.x >> 6;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const long r = r0 + i * 4 + q; const int c = c0 + l;
        t[i * 4 + q][l] = r < rows && c < cols ? to_f32(((const T*)src)[r * ld + c]) : 0.f;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const int c = c0 + i * 4 + q; const long r = r0 + l;
        if (c < cols && r < Rp) gf_emit<T>(dst, plane, (long)c * ldd + r, t[l][i * 4 + q]);
    }
}
// [dg | du] of a 64 x 64 tile of (row, column): rows [N][2 Fp], transposed [2 F][Np], and the tile's column sums
struct GfGrad {
    const void* sg; const void* su; const void* dh; long dh_s; long N; int F, act;
    void* rows; long ldr, plane_r; int Fp; void* cols; long ldc, plane_c; long Np; float* colsum;      // colsum [tiles of N][2 F] or NULL
};
template <class T>
__global__ void __launch_bounds__(256) gf_grad(const GfGrad k) {
    __shared__ float t[2][64][65];
    const long r0 = (long)blockIdx.x * 64; const int c0 = blockIdx.y * 64, l = threadIdx.x & 63, q = threadIdx.x >> 6;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const long r = r0 + i * 4 + q; const int c = c0 + l;
        float dg = 0.f, du = 0.f;
        if (r < k.N && c < k.F) {
            const float g = to_f32(((const T*)k.sg)[r * k.F + c]), u = to_f32(((const T*)k.su)[r * k.F + c]), d = to_f32(((const T*)k.dh)[r * k.dh_s + c]);
            float f, df;
            gf_act_grad(k.act, g, f, df);
            dg = d * u * df; du = d * f;
        }
        t[0][i * 4 + q][l] = dg; t[1][i * 4 + q][l] = du;
        if (r < k.N && c < k.Fp) {
            gf_emit<T>(k.rows, k.plane_r, r * k.ldr + c, dg);
            gf_emit<T>(k.rows, k.plane_r, r * k.ldr + k.Fp + c, du);
        }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const int c = c0 + i * 4 + q; const long r = r0 + l;
        if (c < k.F && r < k.Np) {
            gf_emit<T>(k.cols, k.plane_c, (long)c * k.ldc + r, t[0][l][i * 4 + q]);
            gf_emit<T>(k.cols, k.plane_c, (long)(k.F + c) * k.ldc + r, t[1][l][i * 4 + q]);
        }
    }
    if (k.colsum && threadIdx.x < 128) {
        const int z = threadIdx.x >> 6, c = c0 + l;
        float s = 0.f;
        for (int i = 0; i < 64; ++i) s += t[z][i][l];
        if (c < k.F) k.colsum[(long)blockIdx.x * 2 * k.F + z * k.F + c] = s;
    }
}
// bias gradients: column sums over the row tiles
template <class T>
__global__ void __launch_bounds__(256) gf_bias(const float* part, long R, int F, void* dbg, void* dbu) {
    __shared__ float s[4][64];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, c = blockIdx.x * 64 + lane;
    float acc = 0.f;
    if (c < 2 * F)
        for (long r = w; r < R; r += 4) acc += part[r * 2 * F + c];
    s[w][lane] = acc;
    __syncthreads();
    if (w == 0 && c < 2 * F) {
        const float v = (s[0][lane] + s[1][lane]) + (s[2][lane] + s[3][lane]);
        T* o = (T*)(c < F ? dbg : dbu);
        if (o) o[c < F ? c : c - F] = from_f32<T>(v);
    }
}

// ---- host ----
static int pad64(long n) { return (int)((n + 63) / 64 * 64); }
static bool gf_direct(const refil_gated_ff_desc& d, const void* p, long ld) {
    return d.dtype != REFIL_F32 && d.D % 64 == 0 && ld % 8 == 0 && (uintptr_t)p % 16 == 0;
}
static int gf_planes(int dtype) { return dtype == REFIL_F32 ? 3 : 1; }

// the 256 x 256 tile once its grid covers most of the card, else the 128 x 128 tile, then splits of the reduction
static bool gf_large(long M, long N, int cus) { return cdivl(M, 256) * cdivl(N, 256) >= cus / 2; }
static int gf_cus() {
    static thread_local int cus = 0;
    if (!cus) {
        int dev = 0;
        if (hipGetDevice(&dev) != hipSuccess || hipDeviceGetAttribute(&cus, (hipDeviceAttribute_t)hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || cus <= 0) cus = 256;
    }
    return cus;
}
static int gf_splits(long M, long N, long iters, bool large) {
    const long b = large ? 256 : 128, tiles = cdivl(M, b) * cdivl(N, b), want = 2L * gf_cus();
    if (tiles >= gf_cus()) return 1;
    long s = want / tiles;
    if (s > iters / 8) s = iters / 8;
    if (s > 64) s = 64;
    return s < 1 ? 1 : (int)s;
}

template <class T, bool GATED>
static int gf_launch(GfGemm k, bool large, hipStream_t st, const char* name, double flops, double bytes) {
    typedef typename GfElem<T>::type E;
    const int bm = large ? 256 : 128, half = (large ? 256 : 128) / (GATED ? 2 : 1);
    const long tiles = cdivl(k.M, bm) * cdivl(k.N, half);
    REFIL_CHECK(tiles < (1L << 31), "refil_gated_ff: too many tiles");
    const size_t lds = (size_t)2 * (bm + bm) * 128;
    ProfScope ps(name, flops, bytes, st, nullptr, 0.0, k.pairs > 1 ? flops : 0.0);
    if (large) {
        auto* f = gf_gemm<T, E, 2, 4, 8, 4, GATED>;
        REFIL_HIP(hipFuncSetAttribute((const void*)f, (hipFuncAttribute)hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds));
        hipLaunchKernelGGL(f, dim3(tiles, k.splits), dim3(512), lds, st, k);
    } else {
        auto* f = gf_gemm<T, E, 2, 2, 4, 4, GATED>;
        REFIL_HIP(hipFuncSetAttribute((const void*)f, (hipFuncAttribute)hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds));
        hipLaunchKernelGGL(f, dim3(tiles, k.splits), dim3(256), lds, st, k);
    }
    REFIL_LAUNCH_CHECK();
    return 0;
}

struct GfBump { char* p; size_t n; void* take(size_t b) { char* r = p ? p + n : nullptr; n += (b + 255) / 256 * 256; return r; } };
struct GfFwdWs { void* x; void* wg; void* wu; size_t bytes; };
static GfFwdWs gf_fwd_ws(const refil_gated_ff_desc& d, void* base) {
    GfBump b{(char*)base, 0};
    GfFwdWs w{};
    const size_t es = 2 * gf_planes(d.dtype), Kp = pad64(d.D);
    if (!gf_direct(d, d.x, d.x_stride)) w.x = b.take((size_t)d.N * Kp * es);
    if (!gf_direct(d, d.w_gate, d.w_stride) || !gf_direct(d, d.w_up, d.w_stride)) { w.wg = b.take((size_t)d.F * Kp * es); w.wu = b.take((size_t)d.F * Kp * es); }
    w.bytes = b.n;
    return w;
}
struct GfBwdWs { void* rows; void* cols; void* wt; void* xt; float* colsum; float* part_w; float* part_x; int split_w, split_x; bool large_w, large_x; size_t bytes; };
static GfBwdWs gf_bwd_ws(const refil_gated_ff_desc& d, void* base) {
    GfBump b{(char*)base, 0};
    GfBwdWs w{};
    const size_t es = 2 * gf_planes(d.dtype), Fp = pad64(d.F), Np = pad64(d.N);
    const int pairs = d.dtype == REFIL_F32 ? 6 : 1;
    w.rows = b.take((size_t)d.N * 2 * Fp * es);
    w.cols = b.take((size_t)2 * d.F * Np * es);
    w.wt = b.take((size_t)d.D * 2 * Fp * es);
    w.xt = b.take((size_t)d.D * Np * es);
    w.colsum = (float*)b.take((size_t)cdivl(d.N, 64) * 2 * d.F * 4);
    w.large_x = gf_large(d.N, d.D, gf_cus()); w.large_w = gf_large(2L * d.F, d.D, gf_cus());
    w.split_x = gf_splits(d.N, d.D, (long)pairs * (2 * Fp / 64), w.large_x);
    w.split_w = gf_splits(2L * d.F, d.D, (long)pairs * (Np / 64), w.large_w);
    if (w.split_x > 1) w.part_x = (float*)b.take((size_t)w.split_x * d.N * d.D * 4);
    if (w.split_w > 1) w.part_w = (float*)b.take((size_t)w.split_w * 2 * d.F * d.D * 4);
    w.bytes = b.n;
    return w;
}
static int gf_blocks(long n) { const long b = cdivl(n, 256 * 4); return (int)(b < 1 ? 1 : b > 8192 ? 8192 : b); }

template <class T>
static int gf_forward(const refil_gated_ff_desc& d, hipStream_t st) {
    const GfFwdWs w = gf_fwd_ws(d, d.workspace);
    const int Kp = pad64(d.D);
    GfGemm k{};
    k.pairs = GfElem<T>::planes == 3 ? 6 : 1;
    k.M = (int)d.N; k.N = d.F; k.K = Kp; k.splits = 1;
    k.A = d.x; k.lda = d.x_stride; k.B0 = d.w_gate; k.B1 = d.w_up; k.ldb = d.w_stride;
    if (w.x) {
        hipLaunchKernelGGL((gf_pack<T>), dim3(gf_blocks(d.N * Kp)), dim3(256), 0, st, d.x, (long)d.x_stride, (long)d.N, d.D, Kp, w.x, (long)Kp, (long)d.N * Kp);
        REFIL_LAUNCH_CHECK();
        k.A = w.x; k.lda = Kp; k.planeA = (long)d.N * Kp;
    }
    if (w.wg) {
        hipLaunchKernelGGL((gf_pack<T>), dim3(gf_blocks((long)d.F * Kp)), dim3(256), 0, st, d.w_gate, (long)d.w_stride, (long)d.F, d.D, Kp, w.wg, (long)Kp, (long)d.F * Kp);
        REFIL_LAUNCH_CHECK();
        hipLaunchKernelGGL((gf_pack<T>), dim3(gf_blocks((long)d.F * Kp)), dim3(256), 0, st, d.w_up, (long)d.w_stride, (long)d.F, d.D, Kp, w.wu, (long)Kp, (long)d.F * Kp);
        REFIL_LAUNCH_CHECK();
        k.B0 = w.wg; k.B1 = w.wu; k.ldb = Kp; k.planeB = (long)d.F * Kp;
    }
    k.C0 = d.h; k.ldc = d.h_stride; k.msplit = k.M; k.bias0 = d.b_gate; k.bias1 = d.b_up; k.act = d.act;
    k.save0 = d.saved; k.save1 = d.saved ? (T*)d.saved + d.N * d.F : nullptr;
    const double es = sizeof(T), fl = 4.0 * d.N * d.D * d.F;
    return gf_launch<T, true>(k, gf_large(d.N, 2L * d.F, gf_cus()), st, "gated_ff_fwd", fl, es * ((double)d.N * d.D + 2.0 * d.F * d.D + (d.saved ? 3.0 : 1.0) * d.N * d.F));
}
template <class T>
static int gf_product(GfGemm k, bool large, float* part, hipStream_t st, const char* name, double fl, double bytes) {
    k.partial = part;
    if (int rc = gf_launch<T, false>(k, large, st, name, fl, bytes)) return rc;
    if (k.splits > 1) {
        hipLaunchKernelGGL((gf_reduce<T>), dim3(gf_blocks((long)k.M * k.N)), dim3(256), 0, st, (const float*)part, k.splits, k.M, k.N, k.C0, k.C1, k.ldc, k.msplit);
        REFIL_LAUNCH_CHECK();
    }
    return 0;
}
template <class T>
static int gf_backward(const refil_gated_ff_desc& d, hipStream_t st) {
    const GfBwdWs w = gf_bwd_ws(d, d.workspace);
    const int Fp = pad64(d.F), Np = pad64(d.N), pairs = GfElem<T>::planes == 3 ? 6 : 1;
    const double es = sizeof(T), nf = (double)d.N * d.F;
    GfGrad g{};
    g.sg = d.saved; g.su = (const T*)d.saved + d.N * d.F; g.dh = d.dh; g.dh_s = d.dh_stride; g.N = d.N; g.F = d.F; g.act = d.act;
    g.rows = w.rows; g.ldr = 2L * Fp; g.plane_r = (long)d.N * 2 * Fp; g.Fp = Fp; g.cols = w.cols; g.ldc = Np; g.plane_c = 2L * d.F * Np; g.Np = Np;
    g.colsum = (d.db_gate || d.db_up) ? w.colsum : nullptr;
    {
        ProfScope ps("gated_ff_grad", 20 * nf, (3 + 4) * nf * es, st);
        hipLaunchKernelGGL((gf_grad<T>), dim3(Np / 64, Fp / 64), dim3(256), 0, st, g);
        REFIL_LAUNCH_CHECK();
    }
    if (g.colsum) {
        hipLaunchKernelGGL((gf_bias<T>), dim3(cdiv(2 * d.F, 64)), dim3(256), 0, st, (const float*)w.colsum, (long)(Np / 64), d.F, d.db_gate, d.db_up);
        REFIL_LAUNCH_CHECK();
    }
    typedef typename GfElem<T>::type E;
    hipLaunchKernelGGL((gf_transpose<T>), dim3(Fp / 64, cdiv(d.D, 64)), dim3(256), 0, st, d.w_gate, (long)d.w_stride, (long)d.F, d.D, (long)Fp, w.wt, 2L * Fp, (long)d.D * 2 * Fp);
    REFIL_LAUNCH_CHECK();
    hipLaunchKernelGGL((gf_transpose<T>), dim3(Fp / 64, cdiv(d.D, 64)), dim3(256), 0, st, d.w_up, (long)d.w_stride, (long)d.F, d.D, (long)Fp, (void*)((E*)w.wt + Fp), 2L * Fp, (long)d.D * 2 * Fp);
    REFIL_LAUNCH_CHECK();
    hipLaunchKernelGGL((gf_transpose<T>), dim3(Np / 64, cdiv(d.D, 64)), dim3(256), 0, st, d.x, (long)d.x_stride, (long)d.N, d.D, (long)Np, w.xt, (long)Np, (long)d.D * Np);
    REFIL_LAUNCH_CHECK();
    GfGemm k{};
    k.pairs = pairs;
    k.A = w.rows; k.lda = 2L * Fp; k.planeA = (long)d.N * 2 * Fp; k.B0 = w.wt; k.ldb = 2L * Fp; k.planeB = (long)d.D * 2 * Fp;
    k.M = (int)d.N; k.N = d.D; k.K = 2 * Fp; k.splits = w.split_x; k.C0 = d.dx; k.ldc = d.dx_stride; k.msplit = k.M;
    if (int rc = gf_product<T>(k, w.large_x, w.part_x, st, "gated_ff_dx", 4.0 * nf * d.D, es * (2 * nf + 2.0 * d.F * d.D + (double)d.N * d.D))) return rc;
    k.A = w.cols; k.lda = Np; k.planeA = 2L * d.F * Np; k.B0 = w.xt; k.ldb = Np; k.planeB = (long)d.D * Np;
    k.M = 2 * d.F; k.N = d.D; k.K = Np; k.splits = w.split_w; k.C0 = d.dw_gate; k.C1 = d.dw_up; k.ldc = d.D; k.msplit = d.F;
    return gf_product<T>(k, w.large_w, w.part_w, st, "gated_ff_dw", 4.0 * nf * d.D, es * (2 * nf + 2.0 * d.F * d.D + (double)d.N * d.D));
}
static int gf_check(const refil_gated_ff_desc& d, const char* who) {
    REFIL_CHECK(d.dtype >= REFIL_F32 && d.dtype <= REFIL_F16, "%s: dtype %d is none of REFIL_F32 / REFIL_BF16 / REFIL_F16", who, d.dtype);
    REFIL_CHECK(d.act == REFIL_ACT_SILU || d.act == REFIL_ACT_GELU, "%s: act %d is none of REFIL_ACT_SILU / REFIL_ACT_GELU", who, d.act);
    REFIL_CHECK(d.N >= 0 && d.N <= (1L << 30) && d.D > 0 && d.F > 0 && d.F <= (1 << 20) && d.D <= (1 << 20), "%s: N %lld, D %d, F %d out of range", who, (long long)d.N, d.D, d.F);
    REFIL_CHECK(d.x_stride >= d.D || d.N <= 1, "%s: x_stride %lld below D %d", who, (long long)d.x_stride, d.D);
    REFIL_CHECK(d.w_stride >= d.D, "%s: w_stride %lld below D %d", who, (long long)d.w_stride, d.D);
    return 0;
}

}  // namespace refil

using namespace refil;

extern "C" size_t refil_gated_ff_workspace_bytes(const refil_gated_ff_desc* d, int32_t backward) {
    if (!d || gf_check(*d, "refil_gated_ff_workspace_bytes")) return 0;
    return backward ? gf_bwd_ws(*d, nullptr).bytes : gf_fwd_ws(*d, nullptr).bytes;
}
extern "C" int refil_gated_ff_forward(const refil_gated_ff_desc* d, void* stream) {
    REFIL_CHECK(d, "refil_gated_ff_forward: null desc");
    if (int rc = gf_check(*d, "refil_gated_ff_forward")) return rc;
    if (!d->N) return 0;
    REFIL_CHECK(d->x && d->w_gate && d->w_up && d->h, "refil_gated_ff_forward: x, w_gate, w_up and h are required");
    const size_t need = refil_gated_ff_workspace_bytes(d, 0);
    REFIL_CHECK(!need || (d->workspace && d->workspace_bytes >= need), "refil_gated_ff_forward: workspace of %zu bytes, %zu needed", d->workspace_bytes, need);
    hipStream_t st = (hipStream_t)stream;
    return d->dtype == REFIL_F32 ? gf_forward<float>(*d, st) : d->dtype == REFIL_BF16 ? gf_forward<bf16_t>(*d, st) : gf_forward<f16_t>(*d, st);
}
extern "C" int refil_gated_ff_backward(const refil_gated_ff_desc* d, void* stream) {
    REFIL_CHECK(d, "refil_gated_ff_backward: null desc");
    if (int rc = gf_check(*d, "refil_gated_ff_backward")) return rc;
    REFIL_CHECK(d->N > 0, "refil_gated_ff_backward: no rows");
    REFIL_CHECK(d->x && d->w_gate && d->w_up && d->saved && d->dh && d->dx && d->dw_gate && d->dw_up,
                "refil_gated_ff_backward: x, w_gate, w_up, saved, dh, dx, dw_gate and dw_up are required");
    const size_t need = refil_gated_ff_workspace_bytes(d, 1);
    REFIL_CHECK(d->workspace && d->workspace_bytes >= need, "refil_gated_ff_backward: workspace of %zu bytes, %zu needed", d->workspace_bytes, need);
    hipStream_t st = (hipStream_t)stream;
    return d->dtype == REFIL_F32 ? gf_backward<float>(*d, st) : d->dtype == REFIL_BF16 ? gf_backward<bf16_t>(*d, st) : gf_backward<f16_t>(*d, st);
}
