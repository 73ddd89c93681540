// Gated feed-forward block h = act(x Wg^T + bg) * (x Wu^T + bu), forward and backward (include/refil_hip.h: refil_gated_ff_*).
//
// Every product is C[m][n] = sum_k A(m, k) B(n, k) on v_mfma_f32_16x16x32 (fp32 accumulate), tiles staged through LDS:
//   forward   A = x, B = rows of Wg and Wu interleaved so that one wave holds both projections of a column: bias, activation and product
//             happen in its registers; h (and for training the two pre-activations, fp32) is all that is written
//   backward  one elementwise pass turns the saved pre-activations and dh into [dg | du] (rounded to the type once; fp16: kept in range by a
//             power of two) and the bias sums;
//             dx = [dg | du] [Wg ; Wu] and [dWg ; dWu] = [dg | du]^T x read the operands as they lie in memory: where the reduction index
//             is the row, the LDS tile keeps rows of k and ds_read_b64_tr_b16 hands the matrix core its columns -- nothing is transposed
// fp32 operands are split exactly into three bf16 pieces on their way into LDS and a product runs as six bf16 products (lo hi, hi lo,
// mid mid, mid hi, hi mid, hi hi), as the library's projection GEMMs do.
// Few rows, where the weights' bytes are the cost, and launches of few tiles have a second kernel that reads straight into matrix-core fragments.
//
// Bound by the matrix cores. N 8192, D 2048, F 8192 in bf16: forward with the pre-activations kept 579 us (550 GFLOP, 0.95 PFLOP/s under 671 MB
// of writes), dx 440 us (1.25 PFLOP/s), dw 469 (1.17), the elementwise pass 189 us (940 MB, 5.0 TB/s); a large library product reaches 1.33
// PFLOP/s here. (At the card's steady clock: the first dozen passes take up to 15 % longer.) N 41472, D 128, F 512 in fp32: 122 us forward, 237
// backward, 32.6 GFLOP in all = 91 TFLOP/s of fp32 work (the fp32 instruction's library product: 154 at 8192^3), a fifth of it the elementwise pass.
#include <type_traits>

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
        df = s + v * s * (1.f - s) * (2.f * GF_A) * (1.f + 3.f * GF_B * fminf(v * v, 1e8f));      // (far out s (1 - s) is 0 and v^2 need not be Inf)
    }
}


// ---- the tiled product ----
enum { GF_K = 0, GF_M = 1 };       // an operand's contiguous index: k (rows are m / n) or m / n (rows are k)

__host__ __device__ inline long gf_ldp(int n) { return (n + 3) / 4 * 4; }      // (whole vectors of four: neither side of the partial sums has a ragged end)
struct GfGemm {
    const void* A; long lda;
    const void* B0; const void* B1; long ldb;      // gated: B1 = the up projection; else rows of k at and behind ksplit come from B1
    int M, N, K;
    int a_rows, b_rows;                            // rows that exist of A, of each B (GF_M operands; GF_K: M, N)
    int ksplit;
    int splits; float* partial;                    // splits > 1: fp32 partial sums [splits][M][gf_ldp(N)]
    void* C0; void* C1; long ldc; int msplit, mlim;      // rows m < msplit: row m of C0; the others: row m - msplit of C1; rows at or behind mlim of either are padding
    const void* bias0; const void* bias1; float* save0; float* save1; int act;      // gated epilogue
    const float* unscale;                          // fp16 backward: A holds [dg | du] divided by *unscale, a power of two
};

template <class T>
__device__ __forceinline__ void gf_gated_out(const GfGemm& k, int m, int n, int c, f32x4 ga, f32x4 ua) {
    float g[4], u[4], h[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        g[r] = ga[r]; u[r] = ua[r];
        if (k.bias0 && r < c) g[r] += to_f32(((const T*)k.bias0)[n + r]);
        if (k.bias1 && r < c) u[r] += to_f32(((const T*)k.bias1)[n + r]);
        h[r] = gf_act(k.act, g[r]) * u[r];
    }
    st_raw<T, 4>((T*)k.C0 + (long)m * k.ldc + n, raw_pack<T, 4>(h), c);
    if (k.save0) {
        st_raw<float, 4>(k.save0 + (long)m * k.N + n, raw_pack<float, 4>(g), c);
        st_raw<float, 4>(k.save1 + (long)m * k.N + n, raw_pack<float, 4>(u), c);
    }
}

// wr_split for operands of any finite size. A leading piece that rounds to Inf (the top 0.2 % of the fp32 range) is taken back to the largest bf16
// number of its sign, 0x7F7F or 0xFF7F -- as 16-bit integers the smaller of the two, signed for the positive ones, unsigned for the negative ones --
// and what is left over is below 2^120 and splits exactly.
typedef short gf_s16x2 __attribute__((ext_vector_type(2)));
typedef unsigned short gf_u16x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ void gf_split(float x, float y, unsigned& h, unsigned& m, unsigned& l) {
    const gf_s16x2 p = __builtin_elementwise_min(__builtin_bit_cast(gf_s16x2, wr_pk(x, y)), gf_s16x2{0x7F7F, 0x7F7F});
    h = __builtin_bit_cast(unsigned, __builtin_elementwise_min(__builtin_bit_cast(gf_u16x2, p), gf_u16x2{0xFF7F, 0xFF7F}));
    x -= __uint_as_float(h << 16); y -= __uint_as_float(h & 0xFFFF0000u);
    m = wr_pk(x, y);
    x -= __uint_as_float(m << 16); y -= __uint_as_float(m & 0xFFFF0000u);
    l = wr_pk(x, y);
}
// wr_split, and whether that was needed: `over` becomes Inf. One operation a pair instead of two, for the tiled product, whose vector units the
// split keeps busy (N 4000, D 1024, F 2048: dx and dw 252 + 262 us with the minima in it, 241 + 246 without).
__device__ __forceinline__ void gf_split_watched(float x, float y, unsigned& h, unsigned& m, unsigned& l, float& over) {
    h = wr_pk(x, y);
    x -= __uint_as_float(h << 16); y -= __uint_as_float(h & 0xFFFF0000u);
    over = fmaxf(over, fmaxf(fabsf(x), fabsf(y)));
    m = wr_pk(x, y);
    x -= __uint_as_float(m << 16); y -= __uint_as_float(m & 0xFFFF0000u);
    l = wr_pk(x, y);
}

template <class T> constexpr int GF_P = sizeof(T) == 4 ? 3 : 1;        // 16-bit planes of an operand
template <class T> constexpr int GF_BK = sizeof(T) == 4 ? 32 : 64;
template <class T> struct GfElem { typedef T type; };
template <> struct GfElem<float> { typedef bf16_t type; };

// 64 lanes x 16 bytes of global memory to the 1 KB of LDS behind byte `lds` (wave-uniform), lane order. Inline assembly because the compiler,
// which knows the builtin as a write to LDS, waits for it in front of every transposing read, of the other tile too; nothing but the copy's
// own wait (gf_copies_done, in front of the barrier that hands the tile over) orders it. It has no result registers.
__device__ __forceinline__ void gf_copy16(const void* g, unsigned lds) {
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" : : "v"(g), "s"(lds) : "memory", "m0");
}
__device__ __forceinline__ void gf_copies_done() { asm volatile("s_waitcnt vmcnt(0)" : : : "memory"); }
__device__ __forceinline__ unsigned gf_lds_byte(const char* p) { return (unsigned)(size_t)(const __attribute__((address_space(3))) char*)p; }
static __device__ unsigned gf_zeros[4];        // 16 bytes of zeros that a copy can fetch
typedef short gf_s16x4 __attribute__((ext_vector_type(4)));
// four rows of k, 16 columns: lane i of a 16-lane group supplies columns 4 (i & 3) .. of row i >> 2 and receives column i of the four rows
__device__ __forceinline__ uint2 gf_read_tr(const char* p) {
    return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) gf_s16x4*)p));
}

// Geometry of one operand's LDS tile: ROWS rows of CH chunks of 16 bytes. Which chunk sits in which slot is permuted per row so that the
// fragment reads meet no bank twice (the bank-conflict counter stays 0): GF_K rows (one chunk of 16 rows is read) slot = chunk ^ row bits, of
// rows of four chunks minus row / 4, since a read takes rows 4 i from one half of the lanes with rows 4 i + 12 from the other; GF_M rows
// (32 bytes of eight rows k, k + 1, .. k + 3, k + 8, .. are read) pairs of chunks ^ the row's bits 0, 1 and 3.
template <int LAY, int DIM, int BK> struct GfTile {
    static constexpr int ROWS = LAY == GF_K ? DIM : BK, CH = (LAY == GF_K ? BK : DIM) / 8, BYTES = ROWS * CH * 16;
    __device__ static int swz(int r) { return LAY == GF_K ? (CH == 8 ? (r & 7) : (-(r >> 2) & 3)) : 2 * ((r & 3) | ((r >> 1) & 4)); }
    // fragment of the 16 m (n) behind 16 t, k = 32 kk + 8 (lane / 16) + 0..7
    __device__ static gf_u32x4 frag(const char* tile, int t, int kk, int lane) {
        const int g = lane >> 4, r = lane & 15;
        if constexpr (LAY == GF_K) return *reinterpret_cast<const gf_u32x4*>(tile + ((t * 16 + r) * CH + ((kk * 4 + g) ^ swz(r))) * 16);
        else {
            const int k0 = kk * 32 + g * 8 + (r >> 2);
            const uint2 lo = gf_read_tr(tile + (k0 * CH + ((2 * t) ^ swz(k0))) * 16 + (r & 3) * 8);
            const uint2 hi = gf_read_tr(tile + ((k0 + 4) * CH + ((2 * t) ^ swz(k0 + 4))) * 16 + (r & 3) * 8);
            return gf_u32x4{lo.x, lo.y, hi.x, hi.y};
        }
    }
};

// WM x WN waves, each MT x NT tiles of 16 x 16.
// DIRECT (16-bit, 16-byte aligned rows): global memory goes straight to LDS, two tiles in turn, the next one in flight under the
// products of this one. Otherwise (fp32; odd widths, strides or addresses) it goes through registers -- any alignment, ragged ends filled
// with zeros, fp32 split into its planes -- into one LDS tile, the next one in flight in registers.
template <class T, int LA, int LB, int WM, int WN, int MT, int NT, bool DIRECT, bool GATED>
__global__ void __launch_bounds__(WM * WN * 64, WM * MT == 16 || sizeof(T) == 4 ? 2 : 3) gf_gemm(const GfGemm k) {
    typedef typename GfElem<T>::type E;
    constexpr int P = GF_P<T>, BK = GF_BK<T>, WAVES = WM * WN, THREADS = WAVES * 64, BM = WM * MT * 16, BN = WN * NT * 16, HALF = GATED ? BN / 2 : BN;
    typedef GfTile<LA, BM, BK> TA;
    typedef GfTile<LB, BN, BK> TB;
    constexpr int A_IT = TA::ROWS * TA::CH / THREADS, B_IT = TB::ROWS * TB::CH / THREADS;
    static_assert(!DIRECT || P == 1, "planes are made in registers");
    extern __shared__ __attribute__((aligned(16))) char gf_smem[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int wm = wave / WN, wn = wave % WN;
    const int mt = cdiv(k.M, BM), nt = cdiv(k.N, HALF), total = mt * nt;
    // Consecutive workgroups land on different XCDs (8 of them): each XCD gets a contiguous run of tiles, in panels of 3 rows, so that its
    // L2 holds the panels it reads while many columns are written at a time: N 8192, D 2048, F 8192 with the pre-activations kept took 575 us
    // in panels of 3 and 587 .. 697 us in panels of 1, 2, 4 .. 8, whose writes meet in few memory channels at power-of-two row strides.
    // (One tile per workgroup: walking several with the next one's first block in flight under the outputs
    // measured 517 against 463 us for dx of N 8192, D 2048, F 8192, and no gain elsewhere.)
    int id = blockIdx.x;
    {
        const int per = total / 8, rem = total % 8, xcd = id % 8, pos = id / 8;
        id = xcd * per + min(xcd, rem) + pos;
    }
    constexpr int PR = 3;
    const int panel = id / (PR * nt), prow = min(PR, mt - panel * PR), in_panel = id - panel * PR * nt;
    const int m0 = (panel * PR + in_panel % prow) * BM, n0 = in_panel / prow * HALF;
    const int split = blockIdx.y;
    const int iters = cdiv(k.K, BK), per = cdiv(iters, k.splits), it0 = min(split * per, iters), it1 = min(it0 + per, iters);

    // row n of the (interleaved) B tile -> source and row: NT/2 tiles of the gate, then the same columns of the up projection, per wave
    auto b_row = [&](int r, const T*& src) {
        src = (const T*)k.B0;
        if (!GATED) return n0 + r;
        const int w = r / (NT * 16), j = r % (NT * 16);
        if (j >= NT * 8) src = (const T*)k.B1;
        return n0 + w * NT * 8 + j % (NT * 8);
    };

    f32x4 acc[MT][NT];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

    auto products = [&](const char* a, const char* b) {
#pragma unroll
        for (int kk = 0; kk < BK / 32; ++kk) {
            gf_u32x4 fb[P][NT];
#pragma unroll
            for (int p = 0; p < P; ++p)
#pragma unroll
                for (int j = 0; j < NT; ++j) fb[p][j] = TB::frag(b + p * TB::BYTES, wn * NT + j, kk, lane);
            // D rows = n, columns = m: a lane holds 4 neighbouring n of one m
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                gf_u32x4 fa[P];
#pragma unroll
                for (int p = 0; p < P; ++p) fa[p] = TA::frag(a + p * TA::BYTES, wm * MT + i, kk, lane);
#pragma unroll
                for (int j = 0; j < NT; ++j) {
                    if constexpr (P == 3) {
                        acc[i][j] = gf_mfma<E>(fb[0][j], fa[P - 1], acc[i][j]);
                        acc[i][j] = gf_mfma<E>(fb[P - 1][j], fa[0], acc[i][j]);
                        acc[i][j] = gf_mfma<E>(fb[P / 2][j], fa[P / 2], acc[i][j]);
                        acc[i][j] = gf_mfma<E>(fb[0][j], fa[P / 2], acc[i][j]);
                        acc[i][j] = gf_mfma<E>(fb[P / 2][j], fa[0], acc[i][j]);
                    }
                    acc[i][j] = gf_mfma<E>(fb[0][j], fa[0], acc[i][j]);
                }
            }
        }
    };

    if constexpr (DIRECT) {
        char* const sa = gf_smem; char* const sb = gf_smem + 2 * TA::BYTES;
        const unsigned la = gf_lds_byte(sa), lb = gf_lds_byte(sb);
        const T* pa[A_IT]; const T* pb[B_IT]; int ob[B_IT];      // (ob: a column of B, whose rows change hands at ksplit)
#pragma unroll
        for (int i = 0; i < A_IT; ++i) {
            const int e = (i * WAVES + wave) * 64 + lane, r = e / TA::CH, ch = (e % TA::CH) ^ TA::swz(r);
            if (LA == GF_K) pa[i] = (const T*)k.A + (long)min(m0 + r, k.M - 1) * k.lda + ch * 8;
            else pa[i] = (const T*)k.A + min(m0 + ch * 8, k.M - 8);
        }
#pragma unroll
        for (int i = 0; i < B_IT; ++i) {
            const int e = (i * WAVES + wave) * 64 + lane, r = e / TB::CH, ch = (e % TB::CH) ^ TB::swz(r);
            if (LB == GF_K) {
                const T* src; const int n = b_row(r, src);
                pb[i] = src + (long)min(n, k.N - 1) * k.ldb + ch * 8;
            } else ob[i] = min(n0 + ch * 8, k.N - 8);
        }
        auto stage = [&](int it, int buf) {
            const int k0 = it * BK;
            const bool tail = k0 + BK > k.K;                  // (chunks behind K are zeros of their own; wave-uniform)
#pragma unroll
            for (int i = 0; i < A_IT; ++i) {
                const int e = (i * WAVES + wave) * 64 + lane, r = e / TA::CH;
                const T* p = LA == GF_K ? pa[i] + k0 : pa[i] + (long)min(k0 + r, k.a_rows - 1) * k.lda;
                if (LA == GF_K && tail && k0 + ((e % TA::CH) ^ TA::swz(r)) * 8 >= k.K) p = (const T*)gf_zeros;
                gf_copy16(p, la + buf * TA::BYTES + (i * WAVES + wave) * 1024);
            }
            const T* src = (const T*)k.B0; int kb = k0;
            if (LB == GF_M && k0 >= k.ksplit) { src = (const T*)k.B1; kb -= k.ksplit; }
#pragma unroll
            for (int i = 0; i < B_IT; ++i) {
                const int e = (i * WAVES + wave) * 64 + lane, r = e / TB::CH;
                const T* p = LB == GF_K ? pb[i] + k0 : src + ob[i] + (long)min(kb + r, k.b_rows - 1) * k.ldb;
                if (LB == GF_K && tail && k0 + ((e % TB::CH) ^ TB::swz(r)) * 8 >= k.K) p = (const T*)gf_zeros;
                if (LB == GF_M && kb + BK > k.b_rows && kb + r >= k.b_rows) p = (const T*)gf_zeros;      // (times A's zeros: not another row's Inf)
                gf_copy16(p, lb + buf * TB::BYTES + (i * WAVES + wave) * 1024);
            }
        };
        if (it0 < it1) stage(it0, 0);
        gf_copies_done();
        lds_barrier();
        for (int it = it0; it < it1; ++it) {
            const int buf = (it - it0) & 1;
            if (it + 1 < it1) stage(it + 1, buf ^ 1);
            products(sa + buf * TA::BYTES, sb + buf * TB::BYTES);
            gf_copies_done();
            lds_barrier();
        }
    } else {
        char* const sa = gf_smem; char* const sb = gf_smem + P * TA::BYTES;
        Raw<T> ra[A_IT][8 / VEC_OF<T>], rb[B_IT][8 / VEC_OF<T>];
        constexpr int V = VEC_OF<T>;
        // Eight elements from column `col` of a row of `cols` on. WHOLE (wave-uniform): all there. At an edge a lane reads from where it may -- V
        // columns inside the row, the last row that exists -- and puts right what it got, zeros behind the end (`mend`): no branches, so that the
        // loads leave one behind the other and are waited for once. Rows of fewer than V columns go element by element.
        enum { WHOLE, EDGE, FEW };
        auto fetch = [&](auto way, Raw<T> (&r)[8 / V], const T* row, int col, int cols) {
#pragma unroll
            for (int q = 0; q < 8 / V; ++q) {
                const int c = col + q * V;
                if (way == WHOLE) r[q] = ld_raw<T, V>(row + c, V);
                else if (way == EDGE) r[q] = ld_raw<T, V>(row + min(c, cols - V), V);
                else r[q] = ld_raw<T, V>(row + (c < cols ? c : 0), c < cols ? cols - c : 0);
            }
        };
        auto mend = [&](Raw<T> (&r)[8 / V], int col, int cols, bool in) {
#pragma unroll
            for (int q = 0; q < 8 / V; ++q) {
                const int back = cols >= V ? max(col + q * V - (cols - V), 0) : 0;
                r[q] = raw_down<T, V>(r[q], min(back, V - 1));
#pragma unroll
                for (int w = 0; w < (int)(sizeof(r[q].w) / 4); ++w) r[q].w[w] = in && back < V ? r[q].w[w] : 0u;
            }
        };
        auto load_a = [&](auto way, int k0) {
            const int rows = LA == GF_K ? k.M : min(k.a_rows, k.K), cols = LA == GF_K ? k.K : k.M, r0 = LA == GF_K ? m0 : k0, c0 = LA == GF_K ? k0 : m0;
#pragma unroll
            for (int i = 0; i < A_IT; ++i) {
                const int e = i * THREADS + (int)threadIdx.x, r = e / TA::CH, c = (e % TA::CH) * 8;
                fetch(way, ra[i], (const T*)k.A + (long)(way == WHOLE ? r0 + r : min(r0 + r, rows - 1)) * k.lda, c0 + c, cols);
            }
        };
        auto load_b = [&](auto way, const T* src, int kb) {
            const int rows = LB == GF_K ? k.N : k.b_rows, cols = LB == GF_K ? k.K : k.N, c0 = LB == GF_K ? kb : n0;
#pragma unroll
            for (int i = 0; i < B_IT; ++i) {
                const int e = i * THREADS + (int)threadIdx.x, r = e / TB::CH, c = (e % TB::CH) * 8;
                int row = kb + r;
                if (LB == GF_K) row = b_row(r, src);
                fetch(way, rb[i], src + (long)(way == WHOLE ? row : min(row, rows - 1)) * k.ldb, c0 + c, cols);
            }
        };
        auto load = [&](int it) {
            const int k0 = it * BK;
            typedef std::integral_constant<int, WHOLE> Whole;
            typedef std::integral_constant<int, EDGE> Edge;
            typedef std::integral_constant<int, FEW> Few;
            if (m0 + BM <= k.M && k0 + BK <= (LA == GF_K ? k.K : min(k.a_rows, k.K))) load_a(Whole(), k0);
            else if ((LA == GF_K ? k.K : k.M) >= V) load_a(Edge(), k0);
            else load_a(Few(), k0);
            const T* src = (const T*)k.B0; int kb = k0;
            if (LB == GF_M && k0 >= k.ksplit) { src = (const T*)k.B1; kb -= k.ksplit; }
            if (n0 + HALF <= k.N && kb + BK <= (LB == GF_K ? k.K : k.b_rows)) load_b(Whole(), src, kb);
            else if ((LB == GF_K ? k.K : k.N) >= V) load_b(Edge(), src, kb);
            else load_b(Few(), src, kb);
        };
        // (rows of m or n that are not there need no zeros: what they give is not stored)
        auto fix = [&](int it) {
            const int k0 = it * BK;
            {
                const int rows = min(k.a_rows, k.K), cols = LA == GF_K ? k.K : k.M, c0 = LA == GF_K ? k0 : m0;
                if (c0 + (LA == GF_K ? BK : BM) > cols || (LA == GF_M && k0 + BK > rows)) {
#pragma unroll
                    for (int i = 0; i < A_IT; ++i) {
                        const int e = i * THREADS + (int)threadIdx.x, r = e / TA::CH, c = (e % TA::CH) * 8;
                        mend(ra[i], c0 + c, cols, LA == GF_K || k0 + r < rows);
                    }
                }
            }
            const int kb = LB == GF_M && k0 >= k.ksplit ? k0 - k.ksplit : k0, cols = LB == GF_K ? k.K : k.N, c0 = LB == GF_K ? k0 : n0;
            if (c0 + (LB == GF_K ? BK : BN) > cols || (LB == GF_M && kb + BK > k.b_rows)) {
#pragma unroll
                for (int i = 0; i < B_IT; ++i) {
                    const int e = i * THREADS + (int)threadIdx.x, r = e / TB::CH, c = (e % TB::CH) * 8;
                    mend(rb[i], c0 + c, cols, LB == GF_K || kb + r < k.b_rows);
                }
            }
        };
        float over;
        auto put = [&](auto any_size, char* tile, int bytes, int slot, const Raw<T> (&r)[8 / V]) {
            if constexpr (P == 1) *reinterpret_cast<gf_u32x4*>(tile + slot * 16) = gf_u32x4{r[0].w[0], r[0].w[1], r[0].w[2], r[0].w[3]};
            else {
                unsigned h[4], m[4], l[4];
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const float v0 = raw_get(r[q / 2], 2 * (q & 1)), v1 = raw_get(r[q / 2], 2 * (q & 1) + 1);
                    if constexpr (decltype(any_size)::value) gf_split(v0, v1, h[q], m[q], l[q]);
                    else gf_split_watched(v0, v1, h[q], m[q], l[q], over);
                }
                *reinterpret_cast<gf_u32x4*>(tile + slot * 16) = gf_u32x4{h[0], h[1], h[2], h[3]};
                *reinterpret_cast<gf_u32x4*>(tile + bytes + slot * 16) = gf_u32x4{m[0], m[1], m[2], m[3]};
                *reinterpret_cast<gf_u32x4*>(tile + 2 * bytes + slot * 16) = gf_u32x4{l[0], l[1], l[2], l[3]};
            }
        };
        if (it0 < it1) load(it0);
        for (int it = it0; it < it1; ++it) {
            fix(it);
            lds_barrier();                  // the products of the tile before have been read
            auto put_all = [&](auto any_size) {
#pragma unroll
                for (int i = 0; i < A_IT; ++i) {
                    const int e = i * THREADS + (int)threadIdx.x, r = e / TA::CH;
                    put(any_size, sa, TA::BYTES, r * TA::CH + ((e % TA::CH) ^ TA::swz(r)), ra[i]);
                }
#pragma unroll
                for (int i = 0; i < B_IT; ++i) {
                    const int e = i * THREADS + (int)threadIdx.x, r = e / TB::CH;
                    put(any_size, sb, TB::BYTES, r * TB::CH + ((e % TB::CH) ^ TB::swz(r)), rb[i]);
                }
            };
            over = 0.f;
            put_all(std::false_type());
            if constexpr (P == 3) { if (__any(over == INFINITY)) put_all(std::true_type()); }      // (a lane writes its own slots again)
            lds_barrier();
            if (it + 1 < it1) load(it + 1);
            products(sa, sb);
        }
    }

    // lane: m = lane & 15, n = 4 (lane >> 4) + 0..3 of every tile
    float unscale = 1.f;
    if constexpr (__is_same(T, f16_t) && !GATED) unscale = *k.unscale;
#pragma unroll
    for (int i = 0; i < MT; ++i) {
        const int m = m0 + (wm * MT + i) * 16 + (lane & 15);
        if (m >= k.M) continue;
        if constexpr (GATED) {
#pragma unroll
            for (int j = 0; j < NT / 2; ++j) {
                const int n = n0 + wn * NT * 8 + j * 16 + (lane >> 4) * 4, c = min(max(k.N - n, 0), 4);
                gf_gated_out<T>(k, m, n, c, acc[i][j], acc[i][j + NT / 2]);
            }
        } else {
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                const int n = n0 + (wn * NT + j) * 16 + (lane >> 4) * 4, c = min(max(k.N - n, 0), 4);
                float v[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) v[r] = acc[i][j][r] * unscale;
                if (k.splits > 1) st_raw<float, 4>(k.partial + ((long)split * k.M + m) * gf_ldp(k.N) + n, raw_pack<float, 4>(v), c ? 4 : 0);
                else {
                    const bool first = m < k.msplit;
                    const int row = first ? m : m - k.msplit;
                    if (row < k.mlim) st_raw<T, 4>((T*)(first ? k.C0 : k.C1) + (long)row * k.ldc + n, raw_pack<T, 4>(v), c);
                }
            }
        }
    }
}

// ---- few rows, or few tiles: straight into fragments ----
// A workgroup owns 16 columns of h and 16 MT rows, its eight waves share the reduction; a lane reads 16 neighbouring k (two matrix steps)
// of one weight row, so that a row's reads are whole cache lines -- the order of k inside a product is free as long as both operands share
// it. Up to 64 rows every weight is read once: N 16, D 1024, F 4096 in bf16 5.6 us, 16.8 MB, bound by the launch and one round of latency
// (fp32, N 3, D 3019, F 4313: 104 MB at 3.6 TB/s). With more rows the weights come again from the L2, but eight waves share what one
// workgroup of the tiled kernel would walk alone: taken while that kernel would fill no more than a quarter of the compute units (N 200,
// D 1000, F 1000 in fp32, 32 tiles: 17 against 63 us; N 245, D 257, F 3220, 102 tiles: 33 against 24).
template <class T, int MT>
__global__ void __launch_bounds__(512) gf_skinny(const GfGemm k) {
    typedef typename GfElem<T>::type E;
    constexpr int P = GF_P<T>, V = VEC_OF<T>, Q = 16 / V;
    __shared__ float s_acc[8][2][MT][64][4];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), r = lane & 15, g = lane >> 4;
    const int n0 = blockIdx.x * 16;
    const int mb = blockIdx.y * 16 * MT;
    // (16-bit rows that begin inside a word: 16-byte loads of them cost three times the aligned ones here, where a load's lanes lie in 16 rows --
    // N 170, D 3317, F 791 in bf16 51 us, 25 by whole words, D 3320 17 -- but are the cheaper ones in the tiled kernel, whose lanes follow a row)
    const bool odd_rows = (((size_t)k.A | (size_t)k.B0 | (size_t)k.B1 | (size_t)(k.lda * 2) | (size_t)(k.ldb * 2)) & 3) != 0;
    const T* pg = (const T*)k.B0 + (long)min(n0 + r, k.N - 1) * k.ldb;
    const T* pu = (const T*)k.B1 + (long)min(n0 + r, k.N - 1) * k.ldb;
    f32x4 acc[2][MT];
#pragma unroll
    for (int z = 0; z < 2; ++z)
#pragma unroll
        for (int i = 0; i < MT; ++i) acc[z][i] = f32x4{0.f, 0.f, 0.f, 0.f};
    // (columns of h and rows of x that are not there read the last one: what they give is not stored)
    enum { WHOLE, ODD, RAGGED };
    auto fetch = [&](auto way, Raw<T> (&o)[Q], const T* p, int k0) {
        if constexpr (way == ODD) {
            // Lanes whose 16 elements begin in the middle of a word read the words around them -- the element in front is the row before, or at
            // the first row the storage's: an address that is no multiple of four is not its beginning -- and the last element by itself
            typedef unsigned U4 __attribute__((ext_vector_type(4), aligned(4)));
            p += k0;
            const unsigned odd = ((unsigned)(size_t)p >> 1) & 1;
            const U4 a = *reinterpret_cast<const U4*>(p - odd), b = *reinterpret_cast<const U4*>(p + 8 - odd);
            const unsigned e[9] = {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3], *reinterpret_cast<const unsigned short*>(p + 15)};
#pragma unroll
            for (int i = 0; i < 8; ++i) o[i / 4].w[i % 4] = odd ? (e[i] >> 16) | (e[i + 1] << 16) : e[i];
        } else {
#pragma unroll
            for (int q = 0; q < Q; ++q) {
                const int c = k0 + q * V;
                o[q] = ld_raw<T, V>(p + (way == WHOLE || c < k.K ? c : 0), way == WHOLE ? V : min(max(k.K - c, 0), V));
            }
        }
    };
    auto planes = [&](const Raw<T> (&o)[Q], int half, gf_u32x4 (&f)[P]) {
        if constexpr (P == 1) f[0] = gf_u32x4{o[half].w[0], o[half].w[1], o[half].w[2], o[half].w[3]};
        else {
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                unsigned h, m, l;
                gf_split(raw_get(o[half * 2 + q / 2], 2 * (q & 1)), raw_get(o[half * 2 + q / 2], 2 * (q & 1) + 1), h, m, l);
                f[0][q] = h; f[P / 2][q] = m; f[P - 1][q] = l;
            }
        }
    };
    for (int kb = wave * 64; kb < k.K; kb += 8 * 64) {
        const int k0 = kb + g * 16;
        Raw<T> wg[Q], wu[Q], x[MT][Q];
        auto load = [&](auto way) {
            fetch(way, wg, pg, k0);
            fetch(way, wu, pu, k0);
#pragma unroll
            for (int i = 0; i < MT; ++i) fetch(way, x[i], (const T*)k.A + (long)min(mb + i * 16 + r, k.M - 1) * k.lda, k0);
        };
        if (kb + 64 > k.K) load(std::integral_constant<int, RAGGED>());
        else if (sizeof(T) == 2 && odd_rows) { if constexpr (sizeof(T) == 2) load(std::integral_constant<int, ODD>()); }
        else load(std::integral_constant<int, WHOLE>());
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            gf_u32x4 fg[P], fu[P];
            planes(wg, half, fg);
            planes(wu, half, fu);
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                gf_u32x4 fx[P];
                planes(x[i], half, fx);
                if constexpr (P == 3) {
                    acc[0][i] = gf_mfma<E>(fg[0], fx[P - 1], acc[0][i]); acc[1][i] = gf_mfma<E>(fu[0], fx[P - 1], acc[1][i]);
                    acc[0][i] = gf_mfma<E>(fg[P - 1], fx[0], acc[0][i]); acc[1][i] = gf_mfma<E>(fu[P - 1], fx[0], acc[1][i]);
                    acc[0][i] = gf_mfma<E>(fg[P / 2], fx[P / 2], acc[0][i]); acc[1][i] = gf_mfma<E>(fu[P / 2], fx[P / 2], acc[1][i]);
                    acc[0][i] = gf_mfma<E>(fg[0], fx[P / 2], acc[0][i]); acc[1][i] = gf_mfma<E>(fu[0], fx[P / 2], acc[1][i]);
                    acc[0][i] = gf_mfma<E>(fg[P / 2], fx[0], acc[0][i]); acc[1][i] = gf_mfma<E>(fu[P / 2], fx[0], acc[1][i]);
                }
                acc[0][i] = gf_mfma<E>(fg[0], fx[0], acc[0][i]); acc[1][i] = gf_mfma<E>(fu[0], fx[0], acc[1][i]);
            }
        }
    }
#pragma unroll
    for (int z = 0; z < 2; ++z)
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int q = 0; q < 4; ++q) s_acc[wave][z][i][lane][q] = acc[z][i][q];
    __syncthreads();
    if (wave < MT) {
        f32x4 a[2];
#pragma unroll
        for (int z = 0; z < 2; ++z)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                float t = 0.f;
#pragma unroll
                for (int w = 0; w < 8; ++w) t += s_acc[w][z][wave][lane][q];
                a[z][q] = t;
            }
        const int m = mb + wave * 16 + r, n = n0 + g * 4;
        if (m < k.M) gf_gated_out<T>(k, m, n, min(max(k.N - n, 0), 4), a[0], a[1]);
    }
}

// ---- the elementwise part of the backward ----
// [dg | du] of rows [0, rows_out) (rows behind N and columns behind F are zero: the products read whole 64-blocks of them), rounded to T:
// in 16 bits half a step of each, which the products carry on as they carry x's and the weights'. A workgroup walks `per` rows of 32
// vectors of columns (neighbouring workgroups: neighbouring columns, so that whole rows are in flight) and leaves one partial row of the bias sums, taken before the rounding.
//
// fp16: dg = dh u act' leaves the type's range where dh and the products' results lie in it, so [dg | du] is kept divided by a power of two
// that the products' fp32 sums are multiplied with again (exactly). Almost always that is 1: the pass notes each workgroup's largest finite
// magnitude, and a second launch (gf_regrad) writes everything again, scaled, only where the whole's largest is 61440 or more (Inf), or below 1
// (subnormal numbers, steps of 2^-24, would be felt). One scale for all rows, because a weight gradient adds over them.
struct GfGrad {
    const float* sg; const float* su; const void* dh; long dh_s; long N, rows_out; int F, Fp, act;
    void* out; long ldo; float* colsum; int per;      // colsum [row blocks][2 Fp] or NULL
    float* top; float* unscale;                       // fp16: [workgroups of gf_grad], one number
};
// the workgroup's rows and columns: their [dg | du] times `scale`, their column sums and largest finite magnitude before it
template <class T>
__device__ __forceinline__ void gf_grad_block(const GfGrad& k, int bx, int by, float scale, float (&bg)[VEC_OF<T>], float (&bu)[VEC_OF<T>], float& top) {
    constexpr int V = VEC_OF<T>, CT = 32, RT = 8;
    const int ct = threadIdx.x % CT, rt = threadIdx.x / CT;
    const int c0 = (bx * CT + ct) * V, nv = min(max(k.F - c0, 0), V), np = min(max(k.Fp - c0, 0), V);
    const long r0 = (long)by * k.per, r1 = min(r0 + k.per, k.rows_out);
    for (long r = r0 + rt; r < r1; r += RT) {
        const int n = r < k.N ? nv : 0;
        const long o = r * k.F + c0;
        const auto rd = ld_raw<T, V>((const T*)k.dh + r * k.dh_s + c0, n);
        Raw<float> rg[V / 4], ru[V / 4];
#pragma unroll
        for (int q = 0; q < V / 4; ++q) {
            rg[q] = ld_raw<float, 4>(k.sg + o + q * 4, min(max(n - q * 4, 0), 4));
            ru[q] = ld_raw<float, 4>(k.su + o + q * 4, min(max(n - q * 4, 0), 4));
        }
        float dg[V], du[V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
            float f, df;
            gf_act_grad(k.act, raw_get(rg[i / 4], i % 4), f, df);
            const float d = raw_get(rd, i);
            dg[i] = i < n ? d * raw_get(ru[i / 4], i % 4) * df : 0.f;
            du[i] = i < n ? d * f : 0.f;
            bg[i] += dg[i]; bu[i] += du[i];
            if constexpr (__is_same(T, f16_t)) {
                const float a = fabsf(dg[i]), b = fabsf(du[i]);
                top = fmaxf(top, fmaxf(a < INFINITY ? a : 0.f, b < INFINITY ? b : 0.f));
                dg[i] *= scale; du[i] *= scale;
            }
        }
        T* p = (T*)k.out + r * k.ldo + c0;
        st_raw<T, V>(p, raw_pack<T, V>(dg), np);
        st_raw<T, V>(p + k.Fp, raw_pack<T, V>(du), np);
    }
}
__device__ __forceinline__ float gf_block_max(float v, float (&s)[4]) {
#pragma unroll
    for (int d = 1; d < 64; d *= 2) v = fmaxf(v, __shfl_xor(v, d));
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
    __syncthreads();
    return fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3]));
}
template <class T>
__global__ void __launch_bounds__(256) gf_grad(const GfGrad k) {
    constexpr int V = VEC_OF<T>, CT = 32, RT = 8;
    __shared__ float s[RT][2][CT * V];
    const int ct = threadIdx.x % CT, rt = threadIdx.x / CT;
    float bg[V], bu[V], top = 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i) bg[i] = bu[i] = 0.f;
    gf_grad_block<T>(k, blockIdx.x, blockIdx.y, 1.f, bg, bu, top);
    if constexpr (__is_same(T, f16_t)) {
        __shared__ float s_top[4];
        top = gf_block_max(top, s_top);
        if (threadIdx.x == 0) k.top[(long)blockIdx.y * gridDim.x + blockIdx.x] = top;
    }
    if (!k.colsum) return;
#pragma unroll
    for (int i = 0; i < V; ++i) { s[rt][0][ct * V + i] = bg[i]; s[rt][1][ct * V + i] = bu[i]; }
    __syncthreads();
    for (int e = threadIdx.x; e < 2 * CT * V; e += 256) {
        const int z = e / (CT * V), c = e % (CT * V), col = blockIdx.x * CT * V + c;
        float t = 0.f;
#pragma unroll
        for (int q = 0; q < RT; ++q) t += s[q][z][c];
        if (col < k.F) k.colsum[(long)blockIdx.y * 2 * k.F + z * k.F + col] = t;
    }
}
// every workgroup finds the largest magnitude of all (a maximum: the same in any order) and, if the scale is not 1, walks its share of gf_grad's blocks
__global__ void __launch_bounds__(256) gf_regrad(const GfGrad k, int cols, int blocks) {
    constexpr int V = VEC_OF<f16_t>;
    __shared__ float s_top[4];
    float top = 0.f;
    for (int i = threadIdx.x; i < blocks; i += 256) top = fmaxf(top, k.top[i]);
    top = gf_block_max(top, s_top);
    float scale = 1.f;
    if (top > 0.f && (top < 1.f || top >= 61440.f)) {
        const int e = min(14 - ((int)(__float_as_uint(top) >> 23) - 127), 126);      // [2^14, 2^15) afterwards; far below 2^-112 nearer to 0
        scale = __uint_as_float((unsigned)(127 + e) << 23);
    }
    if (blockIdx.x == 0 && threadIdx.x == 0) *k.unscale = 1.f / scale;               // (a power of two)
    if (scale == 1.f) return;
    float bg[V] = {}, bu[V] = {};
    for (int b = blockIdx.x; b < blocks; b += gridDim.x) gf_grad_block<f16_t>(k, b % cols, b / cols, scale, bg, bu, top);
}
// The end of a backward in one launch: the sums of the split products (dx, then dw) in split order, a thread takes four columns of a row;
// then the bias gradients, 64 columns a workgroup, their partial rows in order.
struct GfFinish { GfGemm dx, dw; int dx_blocks, dw_blocks; const float* colsum; int rows, F; void* dbg; void* dbu; };
template <class T>
__device__ __forceinline__ void gf_reduce(const GfGemm& k, unsigned block, unsigned blocks) {
    const unsigned q = (unsigned)cdiv(k.N, 4), n = (unsigned)k.M * q;          // (fewer tiles than compute units: far below 2^32)
    const long plane = k.M * gf_ldp(k.N);
    for (unsigned e = block * 256 + threadIdx.x; e < n; e += blocks * 256) {
        const int m = (int)(e / q), c0 = (int)(e - (unsigned)m * q) * 4, c = min(k.N - c0, 4);
        const bool first = m < k.msplit;
        const int row = first ? m : m - k.msplit;
        if (row >= k.mlim) continue;
        const float* p = k.partial + m * gf_ldp(k.N) + c0;
        float s[4] = {0.f, 0.f, 0.f, 0.f};
        for (int z = 0; z < k.splits; z += 8) {
            Raw<float> v[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = ld_raw<float>(p + min(z + j, k.splits - 1) * plane, 4);
#pragma unroll
            for (int j = 0; j < 8; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i) s[i] += z + j < k.splits ? raw_get(v[j], i) : 0.f;
        }
        st_raw<T, 4>((T*)(first ? k.C0 : k.C1) + (long)row * k.ldc + c0, raw_pack<T, 4>(s), c);
    }
}
template <class T>
__global__ void __launch_bounds__(256) gf_finish(const GfFinish k) {
    __shared__ float s[4][64];
    if ((int)blockIdx.x < k.dx_blocks) { gf_reduce<T>(k.dx, blockIdx.x, k.dx_blocks); return; }
    if ((int)blockIdx.x < k.dx_blocks + k.dw_blocks) { gf_reduce<T>(k.dw, blockIdx.x - k.dx_blocks, k.dw_blocks); return; }
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, c = ((int)blockIdx.x - k.dx_blocks - k.dw_blocks) * 64 + lane;
    const long ld = 2L * k.F;
    float acc = 0.f;
    if (c < 2 * k.F) {
        int r = w;
        for (; r + 7 * 4 < k.rows; r += 8 * 4) {
            float v[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = k.colsum[(r + j * 4) * ld + c];
#pragma unroll
            for (int j = 0; j < 8; ++j) acc += v[j];
        }
        for (; r < k.rows; r += 4) acc += k.colsum[r * ld + c];
    }
    s[w][lane] = acc;
    __syncthreads();
    if (w == 0 && c < 2 * k.F) {
        T* o = (T*)(c < k.F ? k.dbg : k.dbu);
        if (o) o[c < k.F ? c : c - k.F] = from_f32<T>((s[0][lane] + s[1][lane]) + (s[2][lane] + s[3][lane]));
    }
}

// ---- host ----
static long pad64(long n) { return (n + 63) / 64 * 64; }
static int gf_cus() {
    static thread_local int cus = 0;
    if (!cus) {
        int dev = 0;
        if (hipGetDevice(&dev) != hipSuccess || hipDeviceGetAttribute(&cus, (hipDeviceAttribute_t)hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || cus <= 0) cus = 256;
    }
    return cus;
}
static bool gf_aligned(const refil_gated_ff_desc& d, const void* p, long ld) { return d.dtype != REFIL_F32 && ld % 8 == 0 && (uintptr_t)p % 16 == 0; }
// global memory straight to LDS: 16-byte chunks that never leave their row
static bool gf_direct(const refil_gated_ff_desc& d) {
    return gf_aligned(d, d.x, d.x_stride) && gf_aligned(d, d.w_gate, d.w_stride) && gf_aligned(d, d.w_up, d.w_stride) && d.D % 8 == 0;
}
struct GfPlan { bool direct, large; int splits; };
static GfPlan gf_plan(long M, long N, long K, int bk, bool direct) {
    GfPlan p;
    p.direct = direct;
    p.large = direct && cdivl(M, 256) * cdivl(N, 256) >= gf_cus() / 2;
    const long b = p.large ? 256 : 128, tiles = cdivl(M, b) * cdivl(N, b), iters = cdivl(K, bk);
    long s = tiles >= gf_cus() ? 1 : 2L * gf_cus() / tiles;
    if (s > iters / 4) s = iters / 4;          // (the backward of N 339, D 260, F 294 in fp32: 33 us, 63 with eight blocks each; 1220, 310, 253 in bf16: 34 for 47)
    if (s > 64) s = 64;
    p.splits = s < 1 ? 1 : (int)s;
    return p;
}

template <class T, int LA, int LB, int WM, int WN, int MT, int NT, bool DIRECT, bool GATED>
static int gf_go(const GfGemm& k, hipStream_t st) {
    constexpr int BM = WM * MT * 16, BN = WN * NT * 16, HALF = GATED ? BN / 2 : BN;
    constexpr size_t LDS = (size_t)(DIRECT ? 2 : GF_P<T>) * (GfTile<LA, BM, GF_BK<T>>::BYTES + GfTile<LB, BN, GF_BK<T>>::BYTES);
    const long tiles = cdivl(k.M, BM) * cdivl(k.N, HALF);
    REFIL_CHECK(tiles * k.splits < (1L << 23), "refil_gated_ff: %ld tiles are too many for one launch", tiles);      // (fewer than 2^32 lanes)
    auto* f = gf_gemm<T, LA, LB, WM, WN, MT, NT, DIRECT, GATED>;
    REFIL_HIP(hipFuncSetAttribute((const void*)f, (hipFuncAttribute)hipFuncAttributeMaxDynamicSharedMemorySize, (int)LDS));
    hipLaunchKernelGGL(f, dim3((unsigned)tiles, k.splits), dim3(WM * WN * 64), LDS, st, k);
    REFIL_LAUNCH_CHECK();
    return 0;
}
// Tiles of 32 MT rows instead of 128, where the last of the launch's rounds over the compute units is then so much fuller that fewer rows
// pass in all: N 1537, D 520, F 1366 in fp16 21.2 against 24.3 us (forward, 374 tiles of 96 rows for 286), the backward of N 41472, D 128,
// F 512 in fp32 218 against 222 us (dx, 648 tiles of 64 rows for 324).
template <int MT>
static bool gf_lower(const GfGemm& k, bool gated) {
    const long cols = cdivl(k.N, gated ? 64 : 128);
    return k.splits == 1 && cdivl(cdivl(k.M, 32 * MT) * cols, gf_cus()) * MT < cdivl(cdivl(k.M, 128) * cols, gf_cus()) * 4;
}
template <class T, int LA, int LB, bool GATED>
static int gf_launch(GfGemm k, const GfPlan& p, hipStream_t st, const char* name, double flops, double bytes) {
    ProfScope ps(name, flops, bytes, st, nullptr, 0.0, sizeof(T) == 4 ? flops : 0.0);
    k.splits = p.splits;
    if constexpr (sizeof(T) == 2) {
        if (p.large) return gf_go<T, LA, LB, 2, 4, 8, 4, true, GATED>(k, st);
        if constexpr (LA == GF_K) if (p.direct && gf_lower<3>(k, GATED)) return gf_go<T, LA, LB, 2, 2, 3, 4, true, GATED>(k, st);
        if (p.direct) return gf_go<T, LA, LB, 2, 2, 4, 4, true, GATED>(k, st);
    } else if constexpr (LA == GF_K && !GATED) {
        if (gf_lower<2>(k, GATED)) return gf_go<T, LA, LB, 2, 2, 2, 4, false, GATED>(k, st);
    }
    return gf_go<T, LA, LB, 2, 2, 4, 4, false, GATED>(k, st);
}

static int gf_blocks(long n) { const long b = cdivl(n, 256); return (int)(b < 1 ? 1 : b > 8192 ? 8192 : b); }
struct GfBwdWs { void* grad; float* colsum; float* top; float* unscale; int grad_cols; float* part_x; float* part_w; long Fp, Np; GfPlan px, pw; int row_blocks, per; size_t bytes; };
static GfBwdWs gf_bwd_ws(const refil_gated_ff_desc& d, void* base) {
    char* const p = (char*)base; size_t n = 0;
    auto take = [&](size_t b) { char* r = p ? p + n : nullptr; n += (b + 255) / 256 * 256; return (void*)r; };
    GfBwdWs w{};
    const int bk = d.dtype == REFIL_F32 ? 32 : 64;
    const bool direct = gf_direct(d);
    w.Fp = pad64(d.F); w.Np = pad64(d.N);
    w.grad = take((size_t)w.Np * 2 * w.Fp * (d.dtype == REFIL_F32 ? 4 : 2));
    w.per = (int)(cdivl(cdivl(w.Np, 256), 8) * 8);          // at most 256 partial rows of bias sums, whole rounds of 8 rows
    w.row_blocks = (int)cdivl(w.Np, w.per);
    w.colsum = (float*)take((size_t)w.row_blocks * 2 * d.F * 4);
    w.grad_cols = (int)cdivl(w.Fp, 32 * (d.dtype == REFIL_F32 ? 4 : 8));
    if (d.dtype == REFIL_F16) {
        w.top = (float*)take((size_t)w.grad_cols * w.row_blocks * 4);
        w.unscale = (float*)take(4);
    }
    w.px = gf_plan(d.N, d.D, 2 * w.Fp, bk, direct);
    w.pw = gf_plan(2 * w.Fp, d.D, w.Np, bk, direct);
    if (w.px.splits > 1) w.part_x = (float*)take((size_t)4 * w.px.splits * d.N * gf_ldp(d.D));
    if (w.pw.splits > 1) w.part_w = (float*)take((size_t)4 * w.pw.splits * 2 * w.Fp * gf_ldp(d.D));
    w.bytes = n;
    return w;
}

template <class T>
static int gf_forward(const refil_gated_ff_desc& d, hipStream_t st) {
    GfGemm k{};
    k.A = d.x; k.lda = d.x_stride; k.B0 = d.w_gate; k.B1 = d.w_up; k.ldb = d.w_stride; k.M = (int)d.N; k.N = d.F; k.K = d.D; k.ksplit = 1 << 30; k.splits = 1;
    k.a_rows = k.M; k.b_rows = k.N;
    k.C0 = d.h; k.ldc = d.h_stride; k.bias0 = d.b_gate; k.bias1 = d.b_up; k.act = d.act;
    k.save0 = d.saved; k.save1 = d.saved ? d.saved + d.N * d.F : nullptr;
    const double nf = (double)d.N * d.F, fl = 4 * nf * d.D, by = sizeof(T) * ((double)d.N * d.D + 2.0 * d.F * d.D + nf) + (d.saved ? 8 * nf : 0);
    if (d.N <= 64 || cdivl(d.N, 128) * cdivl(d.F, 64) <= gf_cus() / 4) {
        ProfScope ps("gated_ff_few_rows", fl, by, st, nullptr, 0.0, sizeof(T) == 4 ? fl : 0.0);
        const dim3 grid(cdiv(d.F, 16), cdiv((int)d.N, 64));
        if (d.N <= 16) hipLaunchKernelGGL((gf_skinny<T, 1>), grid, dim3(512), 0, st, k);
        else if (d.N <= 32) hipLaunchKernelGGL((gf_skinny<T, 2>), grid, dim3(512), 0, st, k);
        else hipLaunchKernelGGL((gf_skinny<T, 4>), grid, dim3(512), 0, st, k);
        REFIL_LAUNCH_CHECK();
        return 0;
    }
    GfPlan p = gf_plan(d.N, 2L * d.F, d.D, GF_BK<T>, gf_direct(d));
    p.splits = 1;
    return gf_launch<T, GF_K, GF_K, true>(k, p, st, "gated_ff_fwd", fl, by);
}
template <class T>
static int gf_backward(const refil_gated_ff_desc& d, hipStream_t st) {
    const GfBwdWs w = gf_bwd_ws(d, d.workspace);
    const double es = sizeof(T), nf = (double)d.N * d.F;
    GfGrad g{};
    g.sg = d.saved; g.su = d.saved + d.N * d.F; g.dh = d.dh; g.dh_s = d.dh_stride; g.N = d.N; g.rows_out = w.Np; g.F = d.F; g.Fp = (int)w.Fp; g.act = d.act;
    g.out = w.grad; g.ldo = 2 * w.Fp; g.colsum = (d.db_gate || d.db_up) ? w.colsum : nullptr; g.per = w.per;
    g.top = w.top; g.unscale = w.unscale;
    {
        ProfScope ps("gated_ff_grad", 20 * nf, nf * (8 + 3 * es), st);
        hipLaunchKernelGGL((gf_grad<T>), dim3(w.grad_cols, w.row_blocks), dim3(256), 0, st, g);
        REFIL_LAUNCH_CHECK();
    }
    if constexpr (__is_same(T, f16_t)) {
        const int blocks = w.grad_cols * w.row_blocks;
        ProfScope ps("gated_ff_regrad", 0, 4.0 * blocks, st);
        hipLaunchKernelGGL(gf_regrad, dim3(blocks < 1024 ? blocks : 1024), dim3(256), 0, st, g, w.grad_cols, blocks);
        REFIL_LAUNCH_CHECK();
    }
    GfGemm k{};
    k.A = w.grad; k.lda = 2 * w.Fp; k.B0 = d.w_gate; k.B1 = d.w_up; k.ldb = d.w_stride; k.ksplit = (int)w.Fp;
    k.M = (int)d.N; k.N = d.D; k.K = (int)(2 * w.Fp); k.a_rows = k.M; k.b_rows = d.F; k.C0 = d.dx; k.ldc = d.dx_stride; k.msplit = k.mlim = k.M;
    k.splits = w.px.splits; k.partial = w.part_x; k.unscale = w.unscale;
    GfFinish f{};
    f.dx = k;
    const double fl = 4.0 * nf * d.D, by = es * (2 * nf + 2.0 * d.F * d.D + (double)d.N * d.D);
    if (int rc = gf_launch<T, GF_K, GF_M, false>(k, w.px, st, "gated_ff_dx", fl, by)) return rc;
    k.B0 = d.x; k.ldb = d.x_stride; k.ksplit = 1 << 30;
    k.M = (int)(2 * w.Fp); k.N = d.D; k.K = (int)w.Np; k.a_rows = (int)w.Np; k.b_rows = (int)d.N; k.C0 = d.dw_gate; k.C1 = d.dw_up; k.ldc = d.D; k.msplit = (int)w.Fp; k.mlim = d.F;
    k.splits = w.pw.splits; k.partial = w.part_w;
    f.dw = k;
    if (int rc = gf_launch<T, GF_M, GF_M, false>(k, w.pw, st, "gated_ff_dw", fl, by)) return rc;
    f.dx_blocks = f.dx.splits > 1 ? gf_blocks((long)f.dx.M * f.dx.N / 4) : 0;
    f.dw_blocks = f.dw.splits > 1 ? gf_blocks((long)f.dw.M * f.dw.N / 4) : 0;
    f.colsum = w.colsum; f.rows = w.row_blocks; f.F = d.F; f.dbg = d.db_gate; f.dbu = d.db_up;
    const int blocks = f.dx_blocks + f.dw_blocks + (g.colsum ? cdiv(2 * d.F, 64) : 0);
    if (blocks) {
        ProfScope ps("gated_ff_finish", 0, 4.0 * ((double)f.dx.splits * f.dx.M * f.dx.N + (double)f.dw.splits * f.dw.M * f.dw.N), st);
        hipLaunchKernelGGL((gf_finish<T>), dim3(blocks), dim3(256), 0, st, f);
        REFIL_LAUNCH_CHECK();
    }
    return 0;
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
    return backward ? gf_bwd_ws(*d, nullptr).bytes : 0;
}
extern "C" int refil_gated_ff_forward(const refil_gated_ff_desc* d, void* stream) {
    REFIL_CHECK(d, "refil_gated_ff_forward: null desc");
    if (int rc = gf_check(*d, "refil_gated_ff_forward")) return rc;
    if (!d->N) return 0;
    REFIL_CHECK(d->x && d->w_gate && d->w_up && d->h, "refil_gated_ff_forward: x, w_gate, w_up and h are required");
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
    REFIL_CHECK((uintptr_t)d->workspace % 16 == 0, "refil_gated_ff_backward: workspace must begin on 16 bytes");      // (gf_copy16 reads it)
    hipStream_t st = (hipStream_t)stream;
    return d->dtype == REFIL_F32 ? gf_backward<float>(*d, st) : d->dtype == REFIL_BF16 ? gf_backward<bf16_t>(*d, st) : gf_backward<f16_t>(*d, st);
}
