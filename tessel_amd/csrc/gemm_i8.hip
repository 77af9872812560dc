// Products in 8-bit integers with a scale for each row of X (token) and each
// row of W (channel), the `quant` kernels beside llm/linear and llm/gate_up
// (not .tl kernels):
//   linear   Y[m][n] = f16(SX[m] SW[n] sum_k X[m][k] W[n][k])
//   gate_up  Y[m][f] = f16(silu(g) u), g and u the products with Wg and Wu.
// The sums are v_mfma_i32_16x16x64_i8's, exact in i32 up to K = 131071 (2^14 K
// < 2^31), so no choice of tile, slice or order below changes a bit. The
// scales multiply the sum's f32 value (rounded once above 2^24).
//
// An MFMA operand is 16 bytes a lane here as in the f16 products: lane l holds
// row l % 16 and k 16 (l / 16) .. +15 of a 64-k substep.
#include "common.h"

#include <algorithm>
#include <climits>

namespace {

constexpr int NUM_XCD = 8;
enum Epi8 { Q_LINEAR, Q_SWIGLU };

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef u32x4 u32x4b __attribute__((aligned(1)));

struct Gemm8 {
    const int8_t *X, *W, *W2;        // W2: gate_up's Wu
    const float *SX, *SW, *SW2;
    u16* Y;
    int M, N, K;                     // N: columns of Y
};

// As gemm.hip's: exp as one v_exp_f32, the division as a reciprocal.
TSL_DEV float silu_mul(float g, float u) {
    const float e = __builtin_amdgcn_exp2f(g * -1.4426950408889634f);
    return g * __builtin_amdgcn_rcpf(1.0f + e) * u;
}

// The value of a sum: rounded to f32, times SX, times SW, each product rounded to
// f32 (the asm keeps the last from fusing with the conversion to f16 that may
// follow, which would round once less in some kernels than in others).
TSL_DEV float scaled(int sum, float sx, float sw) {
    float v = (float)sum * sx * sw;
    asm("" : "+v"(v));
    return v;
}

// C tile mapping: a contiguous run of tiles per XCD, walked G tile-rows at a
// time, so that tiles resident together share rows of X and W in its L2.
TSL_DEV void tile_of(int bid, int nwg, int tiles_m, int tiles_n, int G, int& tm, int& tn) {
    int pid = bid;
    if (nwg % NUM_XCD == 0) pid = (bid % NUM_XCD) * (nwg / NUM_XCD) + bid / NUM_XCD;
    const int width = G * tiles_n;
    const int first = (pid / width) * G;
    const int rows = min(tiles_m - first, G);
    tm = first + (pid % width) % rows;
    tn = (pid % width) / rows;
}

// Any K and alignment: 16-byte loads at byte alignment into registers, then LDS.
// Tiles of BM x BN products; gate_up's B tile holds, for each wavefront column, WN / 2 rows of
// Wg and their partners of Wu, so a lane has both sums of an output.
template <int EPI, int BM, int BN>
__global__ __launch_bounds__(256) void gemm_i8_any(Gemm8 a) {
    constexpr bool DUAL = EPI == Q_SWIGLU;
    constexpr int BK = 128, KC = BK / 16;                   // bytes and 16-byte chunks of a tile row
    constexpr int WM = BM / 2, WN = BN / 2, TM = WM / 16, TN = WN / 16;
    constexpr int CA = BM * KC / 256, CB = BN * KC / 256;   // chunks a thread
    constexpr int OUT = DUAL ? BN / 2 : BN;                 // columns of Y a tile
    __shared__ __attribute__((aligned(16))) u32x4 lds[(BM + BN) * KC];
    TSL_POISON(lds);
    auto sw = [](int r) { return (r >> 1) & 7; };
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), t = threadIdx.x;
    const int wm0 = (wave >> 1) * WM, wn0 = (wave & 1) * WN;
    int tm, tn;
    tile_of(blockIdx.x, gridDim.x, (a.M + BM - 1) / BM, (a.N + OUT - 1) / OUT, 8, tm, tn);
    const int m0 = tm * BM, n0 = tn * OUT;
    // Tile row r of B: the row of W (or Wu) it holds.
    auto brow = [&](int r) -> const int8_t* {
        if constexpr (!DUAL) return a.W + (size_t)min(n0 + r, a.N - 1) * a.K;
        const int j = r % WN, n = n0 + (r / WN) * (WN / 2) + j % (WN / 2);
        return (j < WN / 2 ? a.W : a.W2) + (size_t)min(n, a.N - 1) * a.K;
    };
    const int8_t *pa[CA], *pb[CB];
#pragma unroll
    for (int i = 0; i < CA; i++) pa[i] = a.X + (size_t)min(m0 + (i * 256 + t) / KC, a.M - 1) * a.K;
#pragma unroll
    for (int i = 0; i < CB; i++) pb[i] = brow((i * 256 + t) / KC);
    auto chunk = [&](const int8_t* row, int k) {  // 16 k of a row from k on, zeros past K
        if (k + 16 <= a.K) return (u32x4) * reinterpret_cast<const u32x4b*>(row + k);
        u32x4 v = {0, 0, 0, 0};
#pragma unroll
        for (int e = 0; e < 16; e++)
            if (k + e < a.K) v[e >> 2] |= (uint32_t)(uint8_t)row[k + e] << (8 * (e & 3));
        return v;
    };
    i32x4 acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; i++)
#pragma unroll
        for (int j = 0; j < TN; j++) acc[i][j] = i32x4{};
    const int l16 = lane & 15, g16 = lane >> 4;
    for (int k0 = 0; k0 < a.K; k0 += BK) {
        u32x4 ra[CA], rb[CB];
#pragma unroll
        for (int i = 0; i < CA; i++) ra[i] = chunk(pa[i], k0 + 16 * ((i * 256 + t) % KC));
#pragma unroll
        for (int i = 0; i < CB; i++) rb[i] = chunk(pb[i], k0 + 16 * ((i * 256 + t) % KC));
        __syncthreads();
#pragma unroll
        for (int i = 0; i < CA; i++) {
            const int r = (i * 256 + t) / KC, c = (i * 256 + t) % KC;
            lds[r * KC + (c ^ sw(r))] = ra[i];
        }
#pragma unroll
        for (int i = 0; i < CB; i++) {
            const int r = (i * 256 + t) / KC, c = (i * 256 + t) % KC;
            lds[BM * KC + r * KC + (c ^ sw(r))] = rb[i];
        }
        __syncthreads();
#pragma unroll
        for (int st = 0; st < BK / 64; st++) {
            i32x4 av[TM], bv[TN];
#pragma unroll
            for (int i = 0; i < TM; i++) {
                const int r = wm0 + i * 16 + l16;
                av[i] = __builtin_bit_cast(i32x4, lds[r * KC + ((4 * st + g16) ^ sw(r))]);
            }
#pragma unroll
            for (int j = 0; j < TN; j++) {
                const int r = wn0 + j * 16 + l16;
                bv[j] = __builtin_bit_cast(i32x4, lds[BM * KC + r * KC + ((4 * st + g16) ^ sw(r))]);
            }
#pragma unroll
            for (int i = 0; i < TM; i++)
#pragma unroll
                for (int j = 0; j < TN; j++) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(av[i], bv[j], acc[i][j], 0, 0, 0);
        }
    }
    // Lane l of a 16 x 16 tile: column l % 16, rows 4 (l / 16) + r.
    constexpr int TNO = DUAL ? TN / 2 : TN;
#pragma unroll
    for (int j = 0; j < TNO; j++) {
        const int n = n0 + (DUAL ? wn0 / 2 : wn0) + j * 16 + l16;
        if (n >= a.N) continue;
        const float sw1 = a.SW[n], sw2 = DUAL ? a.SW2[n] : 0.0f;
#pragma unroll
        for (int i = 0; i < TM; i++)
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const int m = m0 + wm0 + i * 16 + 4 * g16 + r;
                if (m >= a.M) continue;
                const float sx = a.SX[m];
                float v = scaled(acc[i][j][r], sx, sw1);
                if constexpr (DUAL) v = silu_mul(v, scaled(acc[i][j + TNO][r], sx, sw2));
                a.Y[(size_t)m * a.N + n] = f2h(v);
            }
    }
}

template <int EPI>
int run_gemm8(const Gemm8& a, hipStream_t s) {
    if (a.M == 0 || a.N == 0) return 0;
    constexpr int OUT = EPI == Q_SWIGLU ? 32 : 64;
    const long tiles = (long)((a.M + 63L) / 64) * ((a.N + OUT - 1L) / OUT);
    hipLaunchKernelGGL((gemm_i8_any<EPI, 64, 64>), dim3((unsigned)tiles), dim3(256), 0, s, a);
    return TSL_LAUNCHED("quant product");
}

int check_i8(const TslKernel& k, const char* n) {
    if (k.dim("K") > 131071)
        return tsl_fail(-2, "quant/" + k.name + ": K = " + std::to_string(k.dim("K")) + " exceeds 131071 (sums of 8-bit products in 32 bits)");
    if (k.dim("M") > (1 << 24) || k.dim(n) > (1 << 24))
        return tsl_fail(-2, "quant/" + k.name + ": at most 2^24 rows and columns");
    return 0;
}

}  // namespace

int check_linear_q8(TslKernel& k) { return check_i8(k, "N"); }
int check_gate_up_q8(TslKernel& k) { return check_i8(k, "F"); }

int launch_linear_q8(TslKernel& k, const uint64_t* a, hipStream_t s) {
    return run_gemm8<Q_LINEAR>({P<int8_t>(a[0]), P<int8_t>(a[2]), nullptr, P<float>(a[1]), P<float>(a[3]), nullptr,
                                P<u16>(a[4]), (int)k.dim("M"), (int)k.dim("N"), (int)k.dim("K")}, s);
}

int launch_gate_up_q8(TslKernel& k, const uint64_t* a, hipStream_t s) {
    return run_gemm8<Q_SWIGLU>({P<int8_t>(a[0]), P<int8_t>(a[2]), P<int8_t>(a[4]), P<float>(a[1]), P<float>(a[3]),
                                P<float>(a[5]), P<u16>(a[6]), (int)k.dim("M"), (int)k.dim("F"), (int)k.dim("K")}, s);
}
