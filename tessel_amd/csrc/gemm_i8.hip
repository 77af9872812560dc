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
#include "../../include/tessel.h"
#include "common.h"

#include <algorithm>
#include <climits>
#include <type_traits>

namespace {

constexpr int NUM_XCD = 8;
enum Epi8 { Q_LINEAR, Q_SWIGLU };

typedef int i32x4 __attribute__((ext_vector_type(4)));

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

// 16 k of a row of any alignment from k (a multiple of 16) on, zeros past K: the aligned words that hold them, and
// their shift in a second step (value), so that the loads of later steps can be under way. The fifth
// word is the next lane's first where that lane has the row's next 16 k (lone: it has not), else loaded. A chunk past
// the row's end loads the row's last 16 bytes, so that no word is read that holds no byte of the row.
// (16 bytes at byte alignment take 2 us longer than at 4 in 777 x 1008 x 1155 products, a loaded fifth word of every
// chunk 1.)
struct Row16 {
    u32x4 v;
    uint32_t e = 0;
    TSL_DEV void load(const int8_t* row, int k, int K, bool lone) {
        typedef u32x4 u32x4w __attribute__((aligned(4)));
        if (K >= 16) {
            const int8_t* p = row + min(k, K - 16);
            const uint32_t s = (uint32_t)(uintptr_t)p & 3;
            v = *reinterpret_cast<const u32x4w*>(p - s);
            if (s && (lone || k + 32 > K)) e = *reinterpret_cast<const uint32_t*>(p - s + 16);
        } else {
            v = u32x4{0, 0, 0, 0};
#pragma unroll
            for (int i = 0; i < 15; i++)
                if (k + i < K) v[i >> 2] |= (uint32_t)(uint8_t)row[k + i] << (8 * (i & 3));
        }
    }
    TSL_DEV u32x4 value(const int8_t* row, int k, int K, bool lone) const {
        if (K < 16) return v;
        const uint32_t next = __builtin_amdgcn_mov_dpp((int)v[0], 0x101, 0xf, 0xf, true);  // row_shl:1
        const uint32_t s = (uint32_t)(uintptr_t)(row + min(k, K - 16)) & 3, x = lone || k + 32 > K ? e : next;
        u32x4 w = {__builtin_amdgcn_alignbyte(v[1], v[0], s), __builtin_amdgcn_alignbyte(v[2], v[1], s),
                   __builtin_amdgcn_alignbyte(v[3], v[2], s), __builtin_amdgcn_alignbyte(x, v[3], s)};
        // (No 64-bit shifts: one by an amount that lay in the wavefront's last VGPR gave random results.)
        const int drop = k + 16 - K;  // bytes past K
        if (drop > 0) {
            const bool d8 = drop & 8, d4 = drop & 4;
            const uint32_t a = d8 ? w[2] : w[0], b = d8 ? w[3] : w[1], c = d8 ? 0 : w[2], d = d8 ? 0 : w[3];
            const uint32_t p = d4 ? b : a, q = d4 ? c : b, r = d4 ? d : c, t = d4 ? 0 : d;
            w = u32x4{__builtin_amdgcn_alignbyte(q, p, drop), __builtin_amdgcn_alignbyte(r, q, drop),
                      __builtin_amdgcn_alignbyte(t, r, drop), __builtin_amdgcn_alignbyte(0, t, drop)};
            if (drop >= 16) w = u32x4{0, 0, 0, 0};
        }
        return w;
    }
};

// ---------------------------------------------------------------- aligned rows
// K % 16 == 0 and 16-byte aligned operands: tiles go from global memory into LDS by
// direct buffer loads of 8 rows x 128 bytes (lane i of a load lands at the load's LDS base + 16 i,
// so the swizzle is in which chunk each lane fetches); the resources
// begin at the tile's first row, so operands may be of any size, and rows past the operand's end
// read as zero.
//
// W is the MFMA's A operand and X its B operand, so a lane ends with 4
// consecutive columns of one row of Y a tile; and the rows of W that tile j
// of a wavefront holds are 4 of every 4 TN: row 4 g + r of tile j is W row
// 4 TN g + 4 j + r, so that a lane's tiles together are 4 TN consecutive
// columns, stored 16 bytes at a time. gate_up's wavefronts hold WN / 2
// rows of Wg and the same of Wu, tile by tile, so a lane has both sums of an output.
typedef __attribute__((address_space(3))) void lds_void_t;
constexpr int OOB = 0x7fffffff;  // a byte offset past any range

// s_waitcnt immediate for vmcnt(n) alone (6-bit vmcnt: bits 3:0 and 15:14).
constexpr int vmcnt_imm(int n) { return (n & 15) | ((n >> 4) << 14) | 0x0f70; }

TSL_DEV i32x4 make_rsrc(const void* p, uint32_t bytes) {
    const uint64_t a = reinterpret_cast<uint64_t>(p);
    return i32x4{(int)(uint32_t)a, (int)(uint32_t)((a >> 32) & 0xffff), (int)bytes, 0x00020000};
}

TSL_DEV void load_lds(uint32_t dst, uint32_t off, const i32x4& rs) {
    asm volatile("s_mov_b32 m0, %0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(dst), "v"(off), "s"(rs) : "memory");
}

// Stores a lane's outputs: row m of Y, CNT consecutive columns from n.
template <int CNT>
TSL_DEV void store_cols(u16* Y, int N, int m, int n, const u16 (&v)[CNT]) {
    typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
    typedef u32x4 u32x4h __attribute__((aligned(2)));
    typedef u32x2 u32x2h __attribute__((aligned(2)));
    u16* y = Y + (size_t)m * N + n;
    if (n + CNT <= N) {
        uint32_t w[CNT / 2];
#pragma unroll
        for (int i = 0; i < CNT / 2; i++) w[i] = (uint32_t)v[2 * i] | (uint32_t)v[2 * i + 1] << 16;
        if constexpr (CNT % 8 == 0)
#pragma unroll
            for (int i = 0; i < CNT / 8; i++)
                *reinterpret_cast<u32x4h*>(y + 8 * i) = u32x4{w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]};
        else
#pragma unroll
            for (int i = 0; i < CNT / 4; i++) *reinterpret_cast<u32x2h*>(y + 4 * i) = u32x2{w[2 * i], w[2 * i + 1]};
    } else {
#pragma unroll
        for (int i = 0; i < CNT; i++)
            if (n + i < N) y[i] = v[i];
    }
}

// CNT consecutive steps from n (past N the last one's).
template <int CNT>
TSL_DEV void load_cols(const float* p, int N, int n, float (&v)[CNT]) {
    typedef float4v float4u __attribute__((aligned(4)));
    if (n + CNT <= N) {
#pragma unroll
        for (int i = 0; i < CNT / 4; i++) {
            const float4v t = *reinterpret_cast<const float4u*>(p + n + 4 * i);
#pragma unroll
            for (int e = 0; e < 4; e++) v[4 * i + e] = t[e];
        }
    } else {
#pragma unroll
        for (int c = 0; c < CNT; c++) v[c] = p[min(n + c, N - 1)];
    }
}

// The epilogue of a wavefront's TM x TN tiles: rows m0 + 16 i + l % 16 of Y,
// columns n0 + 4 TNO (l / 16) .. (TNO: tiles of outputs).
template <int EPI, int TM, int TN>
TSL_DEV void store_tiles(const Gemm8& a, int m0, int n0, int lane, const i32x4 (&acc)[TM][TN]) {
    constexpr bool DUAL = EPI == Q_SWIGLU;
    constexpr int TNO = DUAL ? TN / 2 : TN, CNT = 4 * TNO;
    const int n = n0 + CNT * (lane >> 4);
    if (n >= a.N) return;
    float sx[TM], sw[CNT], su[DUAL ? CNT : 1];
#pragma unroll
    for (int i = 0; i < TM; i++) sx[i] = a.SX[min(m0 + 16 * i + (lane & 15), a.M - 1)];
    load_cols<CNT>(a.SW, a.N, n, sw);
    if constexpr (DUAL) load_cols<CNT>(a.SW2, a.N, n, su);
#pragma unroll
    for (int i = 0; i < TM; i++) {
        const int m = m0 + 16 * i + (lane & 15);
        if (m >= a.M) continue;
        u16 v[CNT];
#pragma unroll
        for (int c = 0; c < CNT; c++) {
            float f = scaled(acc[i][c / 4][c % 4], sx[i], sw[c]);
            if constexpr (DUAL) f = silu_mul(f, scaled(acc[i][TNO + c / 4][c % 4], sx[i], su[c]));
            v[c] = f2h(f);
        }
        store_cols<CNT>(a.Y, a.N, m, n, v);
    }
}

// Swizzles of a tile's rows (8 chunks of 16 bytes each): chunk c of row r sits
// at c ^ sw(r), so that the 16 rows of an operand read cover all 16 positions of
// LDS's 256-byte bank window. X reads rows 16 i + l; W (TNO tiles of outputs a wavefront)
// rows 4 TNO (l / 4) + 4 j + l % 4.
TSL_DEV int swx(int r) { return (r >> 1) & 7; }
template <int TNO>
TSL_DEV int sww(int r) { return ((r >> 1) & 1) | (((r / (4 * TNO)) & 3) << 1); }

// Where row r of the W tile comes from: the local output column, and whether it is Wu's.
template <bool DUAL, int WN>
TSL_DEV int w_row(int r) { return DUAL ? (r / WN) * (WN / 2) + r % (WN / 2) : r; }
template <bool DUAL, int WN>
TSL_DEV bool w_up(int r) { return DUAL && r % WN >= WN / 2; }

// Any K and alignment: 16 bytes a lane into registers (Row16), two steps ahead, then LDS.
// 64 x 64 products a workgroup, operands and outputs laid out as the aligned tiles' are; KG groups of 4 wavefronts take
// steps g, g + KG, .. of 128 k through two stages of their own, and their sums are added through LDS at the end (4
// groups where the tiles make one round on the CUs, else 2).
//
// Bound by latency (777 x 1155 x 1001 7.1 us; with loads one step ahead, a load at byte alignment a chunk and
// outputs stored one at a time 9.4), then by the loads, which straddle lines (4001 x 4001 x 1001 71).
template <int EPI, int KG>
__global__ __launch_bounds__(256 * KG) void gemm_i8_any(Gemm8 a) {
    constexpr bool DUAL = EPI == Q_SWIGLU;
    constexpr int BM = 64, BN = 64;
    constexpr int BK = 128, KC = BK / 16;                   // bytes and 16-byte chunks of a tile row
    constexpr int WM = BM / 2, WN = BN / 2, TM = WM / 16, TN = WN / 16, TNO = DUAL ? TN / 2 : TN;
    constexpr int CA = BM * KC / 256, CB = BN * KC / 256;   // chunks a thread
    constexpr int OUT = DUAL ? BN / 2 : BN;                 // columns of Y a tile
    constexpr int STAGE = (BM + BN) * KC;
    __shared__ __attribute__((aligned(16))) u32x4 lds[KG * 2 * STAGE];
    TSL_POISON(lds);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), t = threadIdx.x & 255;
    const int kg = wave >> 2, w4 = wave & 3;
    const int wm0 = (w4 >> 1) * WM, wn0 = (w4 & 1) * WN;
    int tm, tn;
    tile_of(blockIdx.x, gridDim.x, (a.M + BM - 1) / BM, (a.N + OUT - 1) / OUT, 8, tm, tn);
    const int m0 = tm * BM, n0 = tn * OUT, K = a.K;
    u32x4* ring = lds + kg * 2 * STAGE;
    const int8_t *pa[CA], *pb[CB];
    const int c16 = 16 * (t % KC);  // this thread's chunk of every row it loads
#pragma unroll
    for (int i = 0; i < CA; i++) pa[i] = a.X + (size_t)min(m0 + (i * 256 + t) / KC, a.M - 1) * K;
#pragma unroll
    for (int i = 0; i < CB; i++) {
        const int r = (i * 256 + t) / KC;
        pb[i] = (w_up<DUAL, WN>(r) ? a.W2 : a.W) + (size_t)min(n0 + w_row<DUAL, WN>(r), a.N - 1) * K;
    }
    i32x4 acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; i++)
#pragma unroll
        for (int j = 0; j < TN; j++) acc[i][j] = i32x4{};
    const int l16 = lane & 15, g16 = lane >> 4;
    const int xr = wm0 + l16, wr = wn0 + 4 * TNO * (l16 >> 2) + (l16 & 3);  // tile 0's operand rows
    const int rounds = ((K + BK - 1) / BK + KG - 1) / KG;  // (a group past the end multiplies zeros)
    struct Chunks {
        Row16 a[CA], b[CB];
    };
    const bool lone = t % KC == KC - 1;
    auto gload = [&](int round, Chunks& x) {
        const int k = (round * KG + kg) * BK + c16;
#pragma unroll
        for (int i = 0; i < CA; i++) x.a[i].load(pa[i], k, K, lone);
#pragma unroll
        for (int i = 0; i < CB; i++) x.b[i].load(pb[i], k, K, lone);
    };
    auto sstore = [&](int round, const Chunks& x) {
        u32x4* s = ring + (round & 1) * STAGE;
        const int k = (round * KG + kg) * BK + c16;
#pragma unroll
        for (int i = 0; i < CA; i++) {
            const int r = (i * 256 + t) / KC;
            s[r * KC + ((t % KC) ^ swx(r))] = x.a[i].value(pa[i], k, K, lone);
        }
#pragma unroll
        for (int i = 0; i < CB; i++) {
            const int r = (i * 256 + t) / KC;
            s[BM * KC + r * KC + ((t % KC) ^ sww<TNO>(r))] = x.b[i].value(pb[i], k, K, lone);
        }
    };
    // Round q: its stage is written and the other's reads are done; x, the next round's chunks, go to that one, and
    // the round after that is loaded into them.
    auto round = [&](int q, Chunks& x) {
        __syncthreads();
        const u32x4* s = ring + (q & 1) * STAGE;
#pragma unroll
        for (int st = 0; st < BK / 64; st++) {
            i32x4 xv[TM], wv[TN];
#pragma unroll
            for (int i = 0; i < TM; i++)
                xv[i] = __builtin_bit_cast(i32x4, s[(xr + 16 * i) * KC + ((4 * st + g16) ^ swx(xr))]);
#pragma unroll
            for (int j = 0; j < TN; j++) {
                const int r = wr + (j / TNO) * (WN / 2) + 4 * (j % TNO);
                wv[j] = __builtin_bit_cast(i32x4, s[BM * KC + r * KC + ((4 * st + g16) ^ sww<TNO>(r))]);
            }
#pragma unroll
            for (int i = 0; i < TM; i++)
#pragma unroll
                for (int j = 0; j < TN; j++) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wv[j], xv[i], acc[i][j], 0, 0, 0);
        }
        if (q + 1 < rounds) sstore(q + 1, x);
        if (q + 3 < rounds) gload(q + 3, x);
    };
    if (rounds > 0) {
        Chunks x, y;
        gload(0, x);
        if (rounds > 1) gload(1, y);
        sstore(0, x);
        if (rounds > 2) gload(2, x);
        for (int q = 0; q < rounds; q += 2) {
            round(q, y);
            if (q + 1 < rounds) round(q + 1, x);
        }
    }
    __syncthreads();
    i32x4* red = reinterpret_cast<i32x4*>(lds);  // [KG - 1][4 wavefronts][TM TN][64]
    if (kg > 0)
#pragma unroll
        for (int i = 0; i < TM; i++)
#pragma unroll
            for (int j = 0; j < TN; j++) red[(((kg - 1) * 4 + w4) * TM * TN + i * TN + j) * 64 + lane] = acc[i][j];
    __syncthreads();
    if (kg > 0) return;
#pragma unroll
    for (int g = 0; g < KG - 1; g++)
#pragma unroll
        for (int i = 0; i < TM; i++)
#pragma unroll
            for (int j = 0; j < TN; j++) acc[i][j] += red[((g * 4 + w4) * TM * TN + i * TN + j) * 64 + lane];
    store_tiles<EPI, TM, TN>(a, m0 + wm0, n0 + (DUAL ? wn0 / 2 : wn0), lane, acc);
}

// BM x BN tiles, WGM x WGN wavefronts, NS stages of 128 k in a ring. KG groups of wavefronts with a
// ring each take steps g, g + KG, ..; their sums are added through LDS at the end.
template <int EPI, int BM, int BN, int WGM, int WGN, int NS, int KG>
__global__ __launch_bounds__(WGM* WGN* KG * 64, 1) void gemm_i8_tile(Gemm8 a) {
    constexpr bool DUAL = EPI == Q_SWIGLU;
    constexpr int BK = 128, NW = WGM * WGN;
    constexpr int WM = BM / WGM, WN = BN / WGN, TM = WM / 16, TN = WN / 16, TNO = DUAL ? TN / 2 : TN;
    constexpr int OUT = DUAL ? BN / 2 : BN;
    constexpr int LPA = BM / 8 / NW, LPB = BN / 8 / NW, LPS = LPA + LPB;  // 1 KB loads a wavefront a step
    static_assert(BM / 8 % NW == 0 && BN / 8 % NW == 0 && TM >= 1 && TNO >= 1, "tile shape");
    constexpr int STAGE = (BM + BN) * BK;
    static_assert(KG == 1 || (KG - 1) * BM * BN * 4 <= KG * NS * STAGE, "the reduction fits the rings");
    __shared__ __attribute__((aligned(16))) char lds[KG * NS * STAGE];
    TSL_POISON(lds);
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int kg = wave / NW, w = wave % NW;
    const int wm0 = (w / WGN) * WM, wn0 = (w % WGN) * WN;
    int tm, tn;
    tile_of(blockIdx.x, gridDim.x, (a.M + BM - 1) / BM, (a.N + OUT - 1) / OUT, 8, tm, tn);
    const int m0 = tm * BM, n0 = tn * OUT, K = a.K;
    char* ring = lds + kg * NS * STAGE;
    const uint32_t ring_at = (uint32_t)reinterpret_cast<uintptr_t>((lds_void_t*)lds) + kg * NS * STAGE;
    const uint32_t xbytes = (uint32_t)min(BM, a.M - m0) * K, wbytes = (uint32_t)min(OUT, a.N - n0) * K;
    const int8_t *Xt = a.X + (size_t)m0 * K, *Wt = a.W + (size_t)n0 * K, *Wt2 = DUAL ? a.W2 + (size_t)n0 * K : Wt;

    uint32_t offa[LPA], offb[LPB];
    int ka[LPA], kb[LPB];
#pragma unroll
    for (int i = 0; i < LPA; i++) {
        const int r = 8 * (w * LPA + i) + (lane >> 3), c = (lane & 7) ^ swx(r);
        ka[i] = 16 * c;
        offa[i] = (uint32_t)r * K + 16 * c;
    }
#pragma unroll
    for (int i = 0; i < LPB; i++) {
        const int r = 8 * (w * LPB + i) + (lane >> 3), c = (lane & 7) ^ sww<TNO>(r);
        kb[i] = 16 * c;
        offb[i] = (uint32_t)w_row<DUAL, WN>(r) * K + 16 * c;
    }
    // A step's loads into a stage: aim, then load 0 .. LPS - 1 (X's, then W's). Past K (the
    // end of the last step; whole steps of a group that has one less) zeros are loaded.
    i32x4 rx, rw, ru;
    uint32_t dst;
    int kleft;
    auto aim = [&](int step, int stage) {
        const int k0 = step * BK;
        kleft = K - k0;
        const uint32_t skip = min(k0, K);
        rx = make_rsrc(Xt + skip, kleft > 0 ? xbytes - skip : 0);
        rw = make_rsrc(Wt + skip, kleft > 0 ? wbytes - skip : 0);
        ru = DUAL ? make_rsrc(Wt2 + skip, kleft > 0 ? wbytes - skip : 0) : rw;
        dst = ring_at + stage * STAGE;
    };
    auto load = [&](int i) {
        if (i < LPA) load_lds(dst + (w * LPA + i) * 1024, ka[i] < kleft ? offa[i] : (uint32_t)OOB, rx);
        else load_lds(dst + BM * BK + (w * LPB + i - LPA) * 1024, kb[i - LPA] < kleft ? offb[i - LPA] : (uint32_t)OOB,
                      w_up<DUAL, WN>(8 * (w * LPB + i - LPA)) ? ru : rw);
    };
    const int l16 = lane & 15, g16 = lane >> 4;
    const int xr = wm0 + l16, wr = wn0 + 4 * TNO * (l16 >> 2) + (l16 & 3);  // tile 0's operand rows
    auto x_at = [&](int st, int i) { return (uint32_t)((xr + 16 * i) * BK + (((4 * st + g16) ^ swx(xr)) * 16)); };
    auto w_at = [&](int st, int j) {
        const int r = wr + (j / TNO) * (WN / 2) + 4 * (j % TNO);
        return (uint32_t)(BM * BK + r * BK + (((4 * st + g16) ^ sww<TNO>(r)) * 16));
    };
    i32x4 acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; i++)
#pragma unroll
        for (int j = 0; j < TN; j++) acc[i][j] = i32x4{};

    // The ring, software pipelined: step t's second 64 k are read from LDS under its
    // first 64 k's MFMAs, and the next step's first under its second's. Between the
    // two every wavefront holds all of step t in registers and step t + 1 has landed (the
    // barrier), so step t's stage is loaded again, NS - 1 steps ahead. Reads and loads are
    // dealt out between the MFMAs: a wavefront issues in order, and a burst of
    // either would hold the MFMAs behind it.
    const int nsteps = (K + BK - 1) / BK, rounds = (nsteps + KG - 1) / KG;
    constexpr int NM = TM * TN, NR = TM + TN;
    i32x4 xa[TM], wa[TN], xb[TM], wb[TN];
    auto read = [&](int stage, int st, i32x4 (&x)[TM], i32x4 (&v)[TN], int r) {  // the r-th of NR
        const char* sp = ring + stage * STAGE;
        if (r < TN) v[r] = *reinterpret_cast<const i32x4*>(sp + w_at(st, r));
        else x[r - TN] = *reinterpret_cast<const i32x4*>(sp + x_at(st, r - TN));
    };
    auto half = [&](const i32x4 (&x)[TM], const i32x4 (&v)[TN], auto reads, auto loads, int nread, int nload) {
#pragma unroll
        for (int q = 0; q < NM; q++) {
            acc[q / TN][q % TN] = __builtin_amdgcn_mfma_i32_16x16x64_i8(v[q % TN], x[q / TN], acc[q / TN][q % TN], 0, 0, 0);
#pragma unroll
            for (int r = q * nread / NM; r < (q + 1) * nread / NM; r++) reads(r);
#pragma unroll
            for (int r = q * nload / NM; r < (q + 1) * nload / NM; r++) loads(r);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    for (int p = 0; p < NS && p < rounds; p++) {
        aim(p * KG + kg, p);
#pragma unroll
        for (int i = 0; i < LPS; i++) load(i);
    }
    if (rounds >= NS) __builtin_amdgcn_s_waitcnt(vmcnt_imm((NS - 1) * LPS));
    else __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));
    __syncthreads();
#pragma unroll
    for (int r = 0; r < NR; r++) read(0, 0, xa, wa, r);
    int stage = 0;
    auto none = [](int) {};
    auto step = [&](int t, auto more) {
        constexpr bool MORE = decltype(more)::value;
        const int next = stage + 1 == NS ? 0 : stage + 1;
        half(xa, wa, [&](int r) { read(stage, 1, xb, wb, r); }, none, NR, 0);
        __builtin_amdgcn_s_waitcnt(MORE ? vmcnt_imm((NS - 2) * LPS) : vmcnt_imm(0));
        __syncthreads();
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (MORE) {
            aim((t + NS) * KG + kg, stage);
            half(xb, wb, [&](int r) { read(next, 0, xa, wa, r); }, load, NR, LPS);
        } else {
            half(xb, wb, [&](int r) { read(next, 0, xa, wa, r); }, none, NR, 0);
        }
        stage = next;
    };
    int t = 0;
    for (; t + NS < rounds; t++) step(t, std::integral_constant<bool, true>{});
    for (; t + 1 < rounds; t++) step(t, std::integral_constant<bool, false>{});
    half(xa, wa, [&](int r) { read(stage, 1, xb, wb, r); }, none, NR, 0);
    half(xb, wb, none, none, 0, 0);
    if constexpr (KG > 1) {
        i32x4* red = reinterpret_cast<i32x4*>(lds);  // [KG - 1][NW][TM TN][64]
        __syncthreads();
        if (kg > 0)
#pragma unroll
            for (int i = 0; i < TM; i++)
#pragma unroll
                for (int j = 0; j < TN; j++) red[(((kg - 1) * NW + w) * TM * TN + i * TN + j) * 64 + lane] = acc[i][j];
        __syncthreads();
        if (kg > 0) return;
#pragma unroll
        for (int g = 0; g < KG - 1; g++)
#pragma unroll
            for (int i = 0; i < TM; i++)
#pragma unroll
                for (int j = 0; j < TN; j++) acc[i][j] += red[((g * NW + w) * TM * TN + i * TN + j) * 64 + lane];
    }
    store_tiles<EPI, TM, TN>(a, m0 + wm0, n0 + (DUAL ? wn0 / 2 : wn0), lane, acc);
}

// Large products (K % 128 == 0): 256 x 256 tiles as a ping-pong of two groups of
// 4 wavefronts, one of each on every SIMD, in turns between workgroup barriers:
// while one group's MFMAs run back to back from registers, the other reads
// its next step's operands from LDS. gemm_pp16's phases and stages (two of X,
// loaded by group 0; three of W, loaded by group 1 two steps ahead: 160 KB), with 128 k a step.
template <int EPI>
__global__ __launch_bounds__(512, 1) void gemm_i8_pp(Gemm8 a) {
    constexpr bool DUAL = EPI == Q_SWIGLU;
    constexpr int BM = 256, BK = 128;
    constexpr int WM = 128, WN = 64, TM = 8, TN = 4, TNO = DUAL ? 2 : 4, OUT = DUAL ? 128 : 256;
    constexpr int LP = 8;             // 1 KB loads a wavefront a step
    constexpr int TILE = BM * BK;     // bytes of a stage of X (or W)
    constexpr int WBASE = 2 * TILE;
    __shared__ __attribute__((aligned(16))) char lds[5 * TILE];
    TSL_POISON(lds);
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int grp = wave >> 2, w4 = wave & 3;
    const int wm0 = grp * WM, wn0 = w4 * WN;
    int tm, tn;
    tile_of(blockIdx.x, gridDim.x, (a.M + BM - 1) / BM, (a.N + OUT - 1) / OUT, 4, tm, tn);
    const int m0 = tm * BM, n0 = tn * OUT, K = a.K;
    const int l16 = lane & 15, g16 = lane >> 4;
    const uint32_t lds_at = (uint32_t)reinterpret_cast<uintptr_t>((lds_void_t*)lds);
    const uint32_t xbytes = (uint32_t)min(BM, a.M - m0) * K, wbytes = (uint32_t)min(OUT, a.N - n0) * K;
    const int8_t *Xt = a.X + (size_t)m0 * K, *Wt = a.W + (size_t)n0 * K, *Wt2 = DUAL ? a.W2 + (size_t)n0 * K : Wt;

    uint32_t off[LP];
#pragma unroll
    for (int i = 0; i < LP; i++) {
        const int r = 8 * (w4 * LP + i) + (lane >> 3);
        off[i] = grp == 0 ? (uint32_t)r * K + 16 * ((lane & 7) ^ swx(r))
                          : (uint32_t)w_row<DUAL, WN>(r) * K + 16 * ((lane & 7) ^ sww<TNO>(r));
    }
    auto issue = [&](int step, int stage) {
        const int k0 = step * BK;
        auto uniform = [](i32x4 v) {
#pragma unroll
            for (int c = 0; c < 4; c++) v[c] = __builtin_amdgcn_readfirstlane(v[c]);
            return v;
        };
        const i32x4 r0 = uniform(grp == 0 ? make_rsrc(Xt + k0, xbytes - k0) : make_rsrc(Wt + k0, wbytes - k0));
        const i32x4 r1 = uniform(grp == 0 ? r0 : make_rsrc(Wt2 + k0, wbytes - k0));
        const uint32_t dst = __builtin_amdgcn_readfirstlane(lds_at + (grp == 0 ? 0 : WBASE) + stage * TILE + w4 * LP * 1024);
#pragma unroll
        for (int i = 0; i < LP; i++) load_lds(dst + i * 1024, off[i], DUAL && i >= LP / 2 ? r1 : r0);
    };
    static_assert(LP * 8 == WN, "a wavefront of group 1 loads its own rows of W: Wg's, then Wu's");
    const int xr = wm0 + l16, wr = wn0 + 4 * TNO * (l16 >> 2) + (l16 & 3);
    uint32_t x_at[2], w_at[2][TN];
#pragma unroll
    for (int st = 0; st < 2; st++) {
        x_at[st] = (uint32_t)(xr * BK + (((4 * st + g16) ^ swx(xr)) * 16));
#pragma unroll
        for (int j = 0; j < TN; j++) {
            const int r = wr + (j / TNO) * (WN / 2) + 4 * (j % TNO);
            w_at[st][j] = (uint32_t)(WBASE + r * BK + (((4 * st + g16) ^ sww<TNO>(r)) * 16));
        }
    }
    i32x4 xv[2][TM], wv[2][TN];
    auto read_step = [&](int stage, int wstage) {
#pragma unroll
        for (int st = 0; st < 2; st++) {
#pragma unroll
            for (int i = 0; i < TM; i++)
                xv[st][i] = *reinterpret_cast<const i32x4*>(lds + stage * TILE + x_at[st] + i * 16 * BK);
#pragma unroll
            for (int j = 0; j < TN; j++) wv[st][j] = *reinterpret_cast<const i32x4*>(lds + wstage * TILE + w_at[st][j]);
        }
        __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0)
        __builtin_amdgcn_sched_barrier(0);
    };
    i32x4 acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; i++)
#pragma unroll
        for (int j = 0; j < TN; j++) acc[i][j] = i32x4{};
    auto compute = [&]() {
#pragma unroll
        for (int st = 0; st < 2; st++)
#pragma unroll
            for (int i = 0; i < TM; i++)
#pragma unroll
                for (int j = 0; j < TN; j++)
                    acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wv[st][j], xv[st][i], acc[i][j], 0, 0, 0);
        __builtin_amdgcn_sched_barrier(0);
    };
    auto bar = [] {
        __builtin_amdgcn_sched_barrier(0);
        asm volatile("s_barrier" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
    };
    const int nk = K / BK;
    int ws = 0;  // W's stage of step s
    issue(0, 0);
    __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));
    bar();
    if (grp == 0) {
        for (int s = 0; s < nk; s++) {
            if (s + 1 < nk) issue(s + 1, (s + 1) & 1);
            read_step(s & 1, ws);
            bar();
            compute();
            ws = ws == 2 ? 0 : ws + 1;
            __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));
            bar();
        }
    } else {
        if (nk > 1) issue(1, 1);
        bar();
        for (int s = 0; s < nk; s++) {
            read_step(s & 1, ws);
            if (s + 2 < nk) {
                issue(s + 2, ws == 0 ? 2 : ws - 1);
                __builtin_amdgcn_s_waitcnt(vmcnt_imm(LP));
            } else {
                __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));
            }
            bar();
            compute();
            ws = ws == 2 ? 0 : ws + 1;
            if (s + 1 < nk) bar();
        }
    }
    store_tiles<EPI, TM, TN>(a, m0 + wm0, n0 + (DUAL ? wn0 / 2 : wn0), lane, acc);
}

// Few rows (M <= 64): a stream of W. A workgroup of 8 wavefronts has 16 rows of W
// (gate_up: 8 of Wg and their 8 of Wu); wavefront w takes the 128-k steps w, w + 8, ..
// through a ring of D stages of its own (W's 16 rows, X's 16 MT), whole 128-byte
// lines a load, and waits for nobody's loads but its own. The 8 partial
// tiles are added through LDS.
template <int EPI, int MT, int D>
__global__ __launch_bounds__(512) void gemm_i8_skinny(Gemm8 a) {
    constexpr bool DUAL = EPI == Q_SWIGLU;
    constexpr int NWV = 8, BK = 128, STAGE = (16 + 16 * MT) * BK, L = 2 + 2 * MT;  // loads a stage
    constexpr int RING = NWV * D * STAGE, RED = NWV * MT * 1024;
    __shared__ __attribute__((aligned(16))) char lds[RING > RED ? RING : RED];
    TSL_POISON(lds);
    const int lane = threadIdx.x & 63, l16 = lane & 15, g16 = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n0 = blockIdx.x * (DUAL ? 8 : 16), K = a.K;
    const uint32_t wbytes = (uint32_t)min(DUAL ? 8 : 16, a.N - n0) * K, xbytes = (uint32_t)a.M * K;
    const int8_t *Wt = a.W + (size_t)n0 * K, *Wt2 = DUAL ? a.W2 + (size_t)n0 * K : Wt;
    char* ring = lds + wave * D * STAGE;
    const uint32_t ring_at = (uint32_t)reinterpret_cast<uintptr_t>((lds_void_t*)lds) + wave * D * STAGE;
    const int nsteps = (K + BK - 1) / BK, mine = nsteps > wave ? (nsteps - wave + NWV - 1) / NWV : 0;
    auto issue = [&](int u, int stage) {
        const int k0 = (wave + NWV * u) * BK;
        const uint32_t at = ring_at + stage * STAGE;
        const i32x4 rw = make_rsrc(Wt + k0, wbytes - k0), ru = make_rsrc(Wt2 + k0, wbytes - k0), rx = make_rsrc(a.X + k0, xbytes - k0);
#pragma unroll
        for (int i = 0; i < L; i++) {
            const int r = 8 * (i < 2 ? i : i - 2) + (lane >> 3), c = (lane & 7) ^ swx(r);
            const uint32_t off = (uint32_t)(DUAL && i < 2 ? r & 7 : r) * K + 16 * c;
            load_lds(at + i * 1024, k0 + 16 * c < K ? off : (uint32_t)OOB, i >= 2 ? rx : DUAL && i == 1 ? ru : rw);
        }
    };
    for (int u = 0; u < D && u < mine; u++) issue(u, u);
    i32x4 acc[MT];
#pragma unroll
    for (int t = 0; t < MT; t++) acc[t] = i32x4{};
    int stage = 0;
    for (int u = 0; u < mine; u++) {
        const int ahead = min(D - 1, mine - 1 - u);
        if (ahead <= 0) __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));
        else if (ahead == 1) __builtin_amdgcn_s_waitcnt(vmcnt_imm(L));
        else __builtin_amdgcn_s_waitcnt(vmcnt_imm(2 * L));
        asm volatile("" ::: "memory");
        const char* sp = ring + stage * STAGE;
        i32x4 wv[2], xv[2][MT];
#pragma unroll
        for (int st = 0; st < 2; st++) {
            const int c = 16 * ((4 * st + g16) ^ swx(l16));
            wv[st] = *reinterpret_cast<const i32x4*>(sp + l16 * BK + c);
#pragma unroll
            for (int t = 0; t < MT; t++) xv[st][t] = *reinterpret_cast<const i32x4*>(sp + (16 + 16 * t + l16) * BK + c);
        }
#pragma unroll
        for (int st = 0; st < 2; st++)
#pragma unroll
            for (int t = 0; t < MT; t++) acc[t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wv[st], xv[st][t], acc[t], 0, 0, 0);
        // (the operands are in registers before their stage is loaded again)
        __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0)
        asm volatile("" ::: "memory");
        if (u + D < mine) issue(u + D, stage);
        stage = stage + 1 == D ? 0 : stage + 1;
    }
    static_assert(D <= 3, "the waits above");
    // Lane l: W rows 4 (l / 16) + r, row 16 t + l % 16 of X.
    i32x4* red = reinterpret_cast<i32x4*>(lds);  // [MT][wavefront][64]
    __syncthreads();
#pragma unroll
    for (int t = 0; t < MT; t++) red[(t * NWV + wave) * 64 + lane] = acc[t];
    __syncthreads();
    // gate_up: lanes 0 .. 31 hold gate sums, 32 on their up partners.
    for (int t = wave; t < MT; t += NWV) {
        i32x4 s = {0, 0, 0, 0}, u = {0, 0, 0, 0};
#pragma unroll
        for (int w = 0; w < NWV; w++) {
            s += red[(t * NWV + w) * 64 + lane];
            if constexpr (DUAL) u += red[(t * NWV + w) * 64 + (lane | 32)];
        }
        const int m = 16 * t + l16, n = n0 + 4 * g16;
        if (m >= a.M || n >= a.N || (DUAL && g16 >= 2)) continue;
        const float sx = a.SX[m];
        u16 v[4];
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const int nn = min(n + r, a.N - 1);
            float f = scaled(s[r], sx, a.SW[nn]);
            if constexpr (DUAL) f = silu_mul(f, scaled(u[r], sx, a.SW2[nn]));
            v[r] = f2h(f);
        }
        store_cols<4>(a.Y, a.N, m, n, v);
    }
}

template <int EPI, int BM, int BN, int WGM, int WGN, int NS, int KG>
int run_tile(const Gemm8& a, hipStream_t s) {
    constexpr int OUT = EPI == Q_SWIGLU ? BN / 2 : BN;
    const long tiles = (long)((a.M + BM - 1L) / BM) * ((a.N + OUT - 1L) / OUT);
    hipLaunchKernelGGL((gemm_i8_tile<EPI, BM, BN, WGM, WGN, NS, KG>), dim3((unsigned)tiles), dim3(WGM * WGN * KG * 64), 0, s, a);
    return TSL_LAUNCHED("quant product");
}

// The time of a product by each form, in us, from its steps (no form fills the matrix cores or LDS; each is bound by its
// chain of loads, LDS reads and barriers): a step of 128 k costs what it measured on one busy CU, 0.4 of it more with all CUs busy
// (the clock falls), and a product takes as many rounds of them as its tiles need on the CUs:
//   64 x 64 .18 us, 64 x 128 .26, 128 x 128 .37, 256 x 128 .60, 256 x 256 .91, and 3 to 6 us for
// filling, the epilogue and the launch. The skinny form stages 16 rows of W and all of X a block, 54 KB
// a us and CU. Measured / chosen by this, us: linear 65 x 2048 x 5632 64 x 64 10.9
// (256 x 256 44.8), 512 x 4096 x 4096 64 x 128 13.6 (64 x 64 18.0, 128 x 128 17.1), 1024 x 4096
// x 4096 128 x 128 20.7 (256 x 128 26.6), gate_up 512 x 5632 x 2048 256 x 128 16.6 (128 x 128
// 21.2, 256 x 256 24.6), linear 4096 x 4096 x 4096 256 x 256 54.2 (256 x 128 68.6);
// gate_up 32 x 11008 x 4096 64 x 128 16.3 (skinny 22.8), 1 x 5632 x 2048 skinny 4.9 (64 x 64 5.9), linear
// 64 x 2048 x 5632 skinny 6.2 (64 x 64 10.8).
struct Form {
    double step, fixed;
    int bm, out;
};
double form_cost(const Form& f, const Gemm8& a) {
    const double tiles = (double)((a.M + f.bm - 1) / f.bm) * ((a.N + f.out - 1) / f.out), cus = num_cus();
    const double rounds = std::max(1.0, (double)(long)((tiles + cus - 1) / cus)), steps = (a.K + 127) / 128;
    return f.fixed + rounds * steps * f.step * (1.0 + 0.4 * tiles / (rounds * cus));
}

template <int EPI, int MT, int D>
int run_skinny(const Gemm8& a, hipStream_t s) {
    constexpr int ROWS = EPI == Q_SWIGLU ? 8 : 16;
    hipLaunchKernelGGL((gemm_i8_skinny<EPI, MT, D>), dim3((unsigned)((a.N + ROWS - 1) / ROWS)), dim3(512), 0, s, a);
    return TSL_LAUNCHED("quant product");
}

// X's and W's rows (then Wu's) with K no multiple of 16, copied to rows of Kp bytes (whole steps of 128 k), zeros past
// K, for the aligned forms: a wavefront a row, 16 bytes a lane.
__global__ __launch_bounds__(256) void pack_rows_kernel(Gemm8 a, int8_t* __restrict__ out, int Kp, int rows) {
    for (int i = blockIdx.x * 4 + (threadIdx.x >> 6); i < rows; i += gridDim.x * 4) {
        int r = i;
        const int8_t* from = a.X;
        if (r >= a.M) {
            r -= a.M, from = a.W;
            if (r >= a.N) r -= a.N, from = a.W2;
        }
        const int8_t* row = from + (size_t)r * a.K;
        int8_t* to = out + (size_t)i * Kp;
        const bool lone = (threadIdx.x & 15) == 15;
        for (int k = 16 * (threadIdx.x & 63); k < Kp; k += 1024) {
            Row16 x;
            x.load(row, k, a.K, lone);
            *reinterpret_cast<u32x4*>(to + k) = x.value(row, k, a.K, lone);
        }
    }
}

// The aligned forms' costs: the best tile's (K % 128 == 0: the ping-pong too), and the skinny one's (M <= 64).
struct Plan {
    int form;  // 0 .. 4: forms[] below, 5: skinny
    double us;
};
template <int EPI>
Plan plan_aligned(const Gemm8& a) {
    constexpr int HALF = EPI == Q_SWIGLU ? 2 : 1;  // gate_up's tiles hold two rows of W a column
    const Form forms[] = {{0.18, 2.8, 64, 64 / HALF},    {0.26, 3.2, 64, 128 / HALF},   {0.37, 4.0, 128, 128 / HALF},
                          {0.60, 4.2, 256, 128 / HALF}, {0.91, 6.0, 256, 256 / HALF}};
    Plan p = {0, form_cost(forms[0], a)};
    for (int i = 1; i < (a.K % 128 == 0 ? 5 : 4); i++) {
        const double c = form_cost(forms[i], a);
        if (c < p.us) p = {i, c};
    }
    if (a.M <= 64) {
        const double blocks = (a.N + 16 / HALF - 1) / (16 / HALF), kb = (16.0 + (a.M + 15) / 16 * 16) * a.K / 1024;
        const double c = 2.0 + std::max(1.0, blocks / num_cus()) * kb / 54;
        if (c < p.us) p = {5, c};
    }
    return p;
}

template <int EPI>
int run_aligned(const Gemm8& a, hipStream_t s) {
    switch (plan_aligned<EPI>(a).form) {
        case 0: return run_tile<EPI, 64, 64, 2, 2, 4, 2>(a, s);
        case 1: return run_tile<EPI, 64, 128, 2, 2, 3, 2>(a, s);
        case 2: return run_tile<EPI, 128, 128, 2, 4, 4, 1>(a, s);
        case 3: return run_tile<EPI, 256, 128, 4, 2, 3, 1>(a, s);
        case 4: {
            constexpr int OUT = EPI == Q_SWIGLU ? 128 : 256;
            const long tiles = (long)((a.M + 255L) / 256) * ((a.N + OUT - 1L) / OUT);
            hipLaunchKernelGGL(gemm_i8_pp<EPI>, dim3((unsigned)tiles), dim3(512), 0, s, a);
            return TSL_LAUNCHED("quant product");
        }
    }
    switch ((a.M + 15) / 16) {
        case 1: return run_skinny<EPI, 1, 2>(a, s);
        case 2: return run_skinny<EPI, 2, 3>(a, s);
        case 3: return run_skinny<EPI, 3, 2>(a, s);
        default: return run_skinny<EPI, 4, 2>(a, s);
    }
}

// Whether rows of K no multiple of 16 are copied first (into the handle's scratch): gemm_i8_any takes 3.5 us and, a
// step, 0.36 us or its share of 0.55 us a round of the CUs; the copy 3 us and its bytes at 3 TB/s, then the
// aligned forms (us, any / copied: 4001 x 4001 x 1001 71 / 37, 1500 x 2100 x 2001 29.7 / 19.7, 100 x 500 x 9001 27.9
// / 22.1, 777 x 1155 x 1001 7.1 / 9.4, 513 x 3001 x 777 9.9 / 13.2, 1 x 9001 x 4001 17.1 / 22.3).
template <int EPI>
long any_tiles(const Gemm8& a) {
    constexpr int OUT = EPI == Q_SWIGLU ? 32 : 64;
    return (long)((a.M + 63L) / 64) * ((a.N + OUT - 1L) / OUT);
}
template <int EPI>
size_t packed_bytes(Gemm8 a) {
    if (a.K % 16 == 0 || a.M == 0 || a.N == 0) return 0;
    const double steps = (a.K + 127) / 128, any = 3.5 + steps * std::max(0.36, 0.55 * any_tiles<EPI>(a) / num_cus());
    a.K = (a.K + 127) / 128 * 128;
    const size_t bytes = ((size_t)a.M + (EPI == Q_SWIGLU ? 2 : 1) * (size_t)a.N) * a.K;
    return 3.0 + bytes * 2 / 3e6 + plan_aligned<EPI>(a).us < any ? bytes : 0;
}

template <int EPI>
int run_gemm8(Gemm8 a, TslKernel& k, hipStream_t s) {
    if (a.M == 0 || a.N == 0) return 0;
    if (k.scratch) {
        const int kp = (a.K + 127) / 128 * 128, rows = a.M + (EPI == Q_SWIGLU ? 2 : 1) * a.N;
        int8_t* out = reinterpret_cast<int8_t*>(k.scratch);
        hipLaunchKernelGGL(pack_rows_kernel, dim3((unsigned)std::min((rows + 3) / 4, 1 << 16)), dim3(256), 0, s, a, out, kp, rows);
        if (int r = TSL_LAUNCHED("quant product rows")) return r;
        a.X = out, a.W = out + (size_t)a.M * kp, a.W2 = a.W2 ? a.W + (size_t)a.N * kp : nullptr, a.K = kp;
        return run_aligned<EPI>(a, s);
    }
    if (((uint64_t)a.X | (uint64_t)a.W | (uint64_t)a.W2 | (uint64_t)a.K) % 16 == 0 && a.K > 0) return run_aligned<EPI>(a, s);
    const long tiles = any_tiles<EPI>(a);
    if (tiles <= num_cus()) hipLaunchKernelGGL((gemm_i8_any<EPI, 4>), dim3((unsigned)tiles), dim3(1024), 0, s, a);
    else hipLaunchKernelGGL((gemm_i8_any<EPI, 2>), dim3((unsigned)tiles), dim3(512), 0, s, a);
    return TSL_LAUNCHED("quant product");
}

template <int EPI>
int setup_i8(TslKernel& k, const char* n) {
    if (k.dim("K") > 131071)
        return tsl_fail(-2, "quant/" + k.name + ": K = " + std::to_string(k.dim("K")) + " exceeds 131071 (sums of 8-bit products in 32 bits)");
    if (k.dim("M") > (1 << 24) || k.dim(n) > (1 << 24))
        return tsl_fail(-2, "quant/" + k.name + ": at most 2^24 rows and columns");
    // (a launch holds less than 2^32 work-items; 512 of them make 64 x 32 outputs at least)
    if ((k.dim("M") + 63) * (k.dim(n) + 31) >= (1LL << 34)) return tsl_fail(-2, "quant/" + k.name + ": at most 2^34 outputs");
    Gemm8 a{};
    a.M = (int)k.dim("M"), a.N = (int)k.dim(n), a.K = (int)k.dim("K");
    const size_t bytes = packed_bytes<EPI>(a);
    if (!bytes) return 0;
    if (int r = tsl_open()) return r;
    (void)tsl_scratch(k, bytes);  // (no memory for a copy: gemm_i8_any, which needs none)
    return 0;
}

}  // namespace

// What run_gemm8 launches, as tsl_product_form names it.
template <int EPI>
static std::string form_of(const TslKernel& k, const char* n, bool aligned) {
    static const char* const names[] = {"64x64", "64x128", "128x128", "256x128", "256x256"};
    Gemm8 a{};
    a.M = (int)k.dim("M"), a.N = (int)k.dim(n), a.K = (int)k.dim("K");
    if (a.M == 0 || a.N == 0) return "none";
    const bool copied = k.scratch != nullptr;
    if (copied) a.K = (a.K + 127) / 128 * 128;
    else if (!aligned || a.K % 16 || a.K == 0) return any_tiles<EPI>(a) <= num_cus() ? "any 4" : "any 2";
    const int form = plan_aligned<EPI>(a).form;
    return (copied ? "copied " : "") + (form < 5 ? std::string(names[form]) : "skinny " + std::to_string((a.M + 15) / 16 * 16));
}
std::string quant_product_form(const TslKernel& k, bool aligned) {
    return k.name == "linear" ? form_of<Q_LINEAR>(k, "N", aligned) : form_of<Q_SWIGLU>(k, "F", aligned);
}

int setup_linear_q8(TslKernel& k) { return setup_i8<Q_LINEAR>(k, "N"); }
int setup_gate_up_q8(TslKernel& k) { return setup_i8<Q_SWIGLU>(k, "F"); }

int launch_linear_q8(TslKernel& k, const uint64_t* a, hipStream_t s) {
    return run_gemm8<Q_LINEAR>({P<int8_t>(a[0]), P<int8_t>(a[2]), nullptr, P<float>(a[1]), P<float>(a[3]), nullptr,
                                P<u16>(a[4]), (int)k.dim("M"), (int)k.dim("N"), (int)k.dim("K")}, k, s);
}

int launch_gate_up_q8(TslKernel& k, const uint64_t* a, hipStream_t s) {
    return run_gemm8<Q_SWIGLU>({P<int8_t>(a[0]), P<int8_t>(a[2]), P<int8_t>(a[4]), P<float>(a[1]), P<float>(a[3]),
                                P<float>(a[5]), P<u16>(a[6]), (int)k.dim("M"), (int)k.dim("F"), (int)k.dim("K")}, k, s);
}
