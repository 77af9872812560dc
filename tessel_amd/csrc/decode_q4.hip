// Decode attention over the paged cache in 4 bits (quant/decode_attention; not a
// .tl kernel): llm/decode_attention with K and V given as 4-bit codes and a
// pair (lowest value, step) for each token and kv head, value = low + step code.
//   Kc [NP, G, P, D/2]:       byte j of a token: channels 2j (low nibble), 2j + 1
//   Vc [NP, G, P/16, D/2, 16]: the same bytes, 16 tokens of a channel pair together
//   Ks, Vs [NP, G, P, 2]:     (low, step), f16
// With low and step factored out, a score is
//   q . k = step (q . n) + low sum(q)
// and an output sum(p v) = sum((p step) (n - 8)) + sum(p (low + 8 step)), so only small whole
// numbers go through the products (values centred, for sums of codes 0 .. 15 are some 20 times the outputs that
// they cancel to, and round accordingly). A page outside [0, NP) reads as zeros and an
// empty sequence is 0/0 = NaN, as in decode_attention; a length past the table's
// MP P tokens counts as MP P.
#include "common.h"

#include <algorithm>
#include <climits>

int check_cache_q4(const TslKernel& k);

namespace {

constexpr float LOG2E = 1.4426950408889634f;

struct Q4Args {
    const u16* Q;
    const uint8_t *Kc, *Vc;
    const u16 *Ks, *Vs;
    const int *table, *lens;
    u16* O;
    float* part;  // [B][G][NCH][QPG][2 + D]: m, l, acc
    int B, H, G, NP, P, MP, NCH;
    int CT;       // tokens per chunk (a multiple of 256)
    int pshift;   // log2(P)
    bool wide;    // one chunk a sequence, 8 wavefronts
    int first;    // sequences are taken by length, the first of them longest first, then shortest first (0: in order)
    float c2;     // scale log2(e)
};

// The page of token t of sequence b (-1: outside the pool).
TSL_DEV int page_of(const Q4Args& a, int b, int t) {
    const int page = a.table[(long)b * a.MP + t / a.P];
    return page >= 0 && page < a.NP ? page : -1;
}

// Tokens of sequence b: lens[b], at most what its table holds.
TSL_DEV int tokens_of(const Q4Args& a, int b) { return min(max(a.lens[b], 0), a.MP * a.P); }

// A workgroup per (sequence, kv head, chunk of CT tokens), 256 tokens at a time:
// a thread scores one token for the QPG query heads, then a thread per
// (channel pair, block of 16 tokens) adds its share of the values.
template <int D, int QPG>
__global__ __launch_bounds__(256) void decode_q4_any(Q4Args a) {
    constexpr int D2 = D / 2, NG = 256 / D2;  // groups of blocks
    __shared__ float qs[QPG][D], qsum[QPG], sc[QPG][256];
    __shared__ float mrun[QPG], lrun[QPG], keep[QPG], lowsum[QPG], part[4][QPG][2], red[NG][D];
    TSL_POISON(qs); TSL_POISON(sc); TSL_POISON(part); TSL_POISON(red);
    const int tid = threadIdx.x;
    const int c = blockIdx.x / (a.B * a.G);
    const long bg = blockIdx.x % (a.B * a.G);
    const int g = bg % a.G, b = bg / a.G;
    const int n = tokens_of(a, b);
    if (n <= c * a.CT) {
        if (c == 0)  // an empty sequence: 0 / 0
            for (int i = tid; i < QPG * D; i += 256) a.O[((long)b * a.H + g * QPG) * D + i] = 0x7e00;
        return;
    }
    const int t_lo = c * a.CT, t_hi = min(n - t_lo, a.CT) + t_lo;
    for (int i = tid; i < QPG * D; i += 256) qs[i / D][i % D] = h2f(a.Q[((long)b * a.H + g * QPG) * D + i]);
    if (tid < QPG) mrun[tid] = -INFINITY, lrun[tid] = 0.0f, lowsum[tid] = 0.0f;
    __syncthreads();
    if (tid < QPG) {
        float s = 0.0f;
        for (int d = 0; d < D; d++) s += qs[tid][d];
        qsum[tid] = s;
    }
    __syncthreads();
    const int j = tid % D2, grp = tid / D2;
    float acc[QPG][2];
#pragma unroll
    for (int i = 0; i < QPG; i++) acc[i][0] = acc[i][1] = 0.0f;
    for (int done = 0; done < t_hi - t_lo; done += 256) {
        const int t0 = t_lo + done, t = t0 + tid;
        const bool live = tid < t_hi - t0;
        const int page = live ? page_of(a, b, t) : -1;
        float s[QPG], vlow = 0.0f, vstep = 0.0f;
#pragma unroll
        for (int i = 0; i < QPG; i++) s[i] = live ? 0.0f : -INFINITY;
        if (page >= 0) {
            const long at = ((long)page * a.G + g) * a.P + t % a.P;
            const uint8_t* kp = a.Kc + at * D2;
            for (int e = 0; e < D2; e++) {
                const float n0 = kp[e] & 15, n1 = kp[e] >> 4;
#pragma unroll
                for (int i = 0; i < QPG; i++) s[i] += qs[i][2 * e] * n0 + qs[i][2 * e + 1] * n1;
            }
            const float low = h2f(a.Ks[2 * at]), step = h2f(a.Ks[2 * at + 1]);
#pragma unroll
            for (int i = 0; i < QPG; i++) s[i] = (s[i] * step + low * qsum[i]) * a.c2;
            vstep = h2f(a.Vs[2 * at + 1]);
            vlow = __builtin_fmaf(8.0f, vstep, h2f(a.Vs[2 * at]));
        }
#pragma unroll
        for (int i = 0; i < QPG; i++) sc[i][tid] = s[i];
        __syncthreads();
        // A wavefront per query head: the running maximum, and what the earlier sums are scaled by.
        for (int i = tid >> 6; i < QPG; i += 4) {
            float m = -INFINITY;
            for (int x = tid & 63; x < 256; x += 64) m = fmaxf(m, sc[i][x]);
            m = fmaxf(mrun[i], wave_max(m));
            if ((tid & 63) == 0) {
                keep[i] = __builtin_amdgcn_exp2f(mrun[i] - m);
                mrun[i] = m;
            }
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < QPG; i++) {
            const float p = __builtin_amdgcn_exp2f(s[i] - mrun[i]);
            sc[i][tid] = p * vstep;
            const float l = wave_sum(p), lw = wave_sum(p * vlow);
            if ((tid & 63) == 0) part[tid >> 6][i][0] = l, part[tid >> 6][i][1] = lw;
        }
        __syncthreads();
        if (tid < QPG) {
            float l = 0.0f, lw = 0.0f;
            for (int w = 0; w < 4; w++) l += part[w][tid][0], lw += part[w][tid][1];
            lrun[tid] = lrun[tid] * keep[tid] + l;
            lowsum[tid] = lowsum[tid] * keep[tid] + lw;
        }
#pragma unroll
        for (int i = 0; i < QPG; i++) acc[i][0] *= keep[i], acc[i][1] *= keep[i];
        for (int blk = grp; blk < 16; blk += NG) {
            if (16 * blk >= t_hi - t0) break;
            const int tb = t0 + 16 * blk, pg = page_of(a, b, tb);
            if (pg < 0) continue;
            const u32x4 w = *reinterpret_cast<const u32x4*>(
                a.Vc + ((((long)pg * a.G + g) * (a.P / 16) + tb % a.P / 16) * D2 + j) * 16);
            for (int x = 0; x < 16; x++) {
                const uint32_t v = (w[x >> 2] >> (8 * (x & 3))) & 255;
                const float n0 = (int)(v & 15) - 8, n1 = (int)(v >> 4) - 8;
#pragma unroll
                for (int i = 0; i < QPG; i++) acc[i][0] += sc[i][16 * blk + x] * n0, acc[i][1] += sc[i][16 * blk + x] * n1;
            }
        }
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < QPG; i++) {
        __syncthreads();
        red[grp][2 * j] = acc[i][0];
        red[grp][2 * j + 1] = acc[i][1];
        __syncthreads();
        if (tid < D) {
            float v = lowsum[i];
            for (int x = 0; x < NG; x++) v += red[x][tid];
            if (a.NCH == 1) {
                a.O[((long)b * a.H + g * QPG + i) * D + tid] = f2h(v / lrun[i]);
            } else {
                float* p = a.part + ((bg * a.NCH + c) * QPG + i) * (2 + D);
                if (tid == 0) p[0] = mrun[i], p[1] = lrun[i];
                p[2 + tid] = v;
            }
        }
    }
}

// ---------------------------------------------------------------- the matrix-core form
// D = 32, 64 or 128. A workgroup of NW wavefronts has one (sequence, kv head, chunk of at most
// CHUNK_MAX tokens); wavefront w takes the 64-token tiles w, w + NW, .. of the chunk, the next
// tile's loads in flight. All of a tile goes from memory into registers in the operands' own shapes:
//
//   S^T = K Q^T, four tiles of 16 tokens x 16 query heads (v_mfma_f32_16x16x32_f16): row i of tile a is
//   token 4 a + i % 4 of block i / 4 (a tile of 64 tokens is 4 blocks of 16), so that lane (head, g) ends with
//   the 16 tokens of block g in order; its 16 bytes of V's layout are those tokens of a channel pair:
//   O^T += V^T P^T, 16 channels x 16 heads a tile, channels of one parity, tokens 8 u .. 8 u + 7 of every block a step.
//
// A key's code needs no conversion: in an f16's bits 9 .. 6 it is the subnormal n 2^-18, two operations for two codes.
// (In bits 3 .. 0, n 2^-24, one operation less for eight: but a product is aligned by its operands' exponents, a
// subnormal's being 2^-14, and what lies 24 bits below the largest one is cut off. Sums of such codes were off by 19 times
// 2^-23 of their largest term, one way, these by 0.2: 64 x 128-4096 tokens were 5e-5 off before the output's rounding,
// 0.17 of the outputs another f16 than the exact one's.) A value's code goes under the exponent of 1024, from
// where one operation takes it to n - 8. q is scaled by a power of two into f16's middle. step and low enter in f32:
// u = step (q . n) + low sum(q); p step is split into two f16, so a probability keeps 22 bits (beside a step up to 2^16 times
// its token's; a further one leaves it those above 2^-38 of that step).
//
// Bound by memory for long caches (64 x 4096 tokens, 8 kv heads of 128: 5.4 TB/s), by latency for short ones; VALU (about 20
// operations a token and query head, in packed lanes, and 17 for 8 codes of keys and 8 of values) is not far below.
constexpr int TILE = 64;
constexpr int CHUNK_MAX = 4096;  // tokens of a chunk, at most (their table entries are held in LDS)
constexpr int RANKED = 512;      // sequences taken by length, at most

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef u32x4 u32x4u __attribute__((aligned(2)));

template <int W>
struct Words {  // a lane's W words of a row
    uint32_t w[W];
    TSL_DEV void load(const uint8_t* p) {
        if constexpr (W == 4) {
            const u32x4 v = *reinterpret_cast<const u32x4*>(p);
            w[0] = v[0], w[1] = v[1], w[2] = v[2], w[3] = v[3];
        } else if constexpr (W == 2) {
            const u32x2 v = *reinterpret_cast<const u32x2*>(p);
            w[0] = v[0], w[1] = v[1];
        } else {
            w[0] = *reinterpret_cast<const uint32_t*>(p);
        }
    }
};

// f16 pairs of a word's codes: low nibbles of bytes (0, 2), (1, 3), then high nibbles; n 2^-18, and n - 8.
TSL_DEV void nibbles(uint32_t w, uint32_t (&lo)[2], uint32_t (&hi)[2]) {
    constexpr uint32_t M = 0x03c003c0u;
    lo[0] = (w << 6) & M, lo[1] = (w >> 2) & M;
    hi[0] = (w << 2) & M, hi[1] = (w >> 6) & M;
}
// (big: 1024 twice, in a VGPR, for one v_and_or_b32 takes one scalar operand.)
TSL_DEV void centred(uint32_t w, uint32_t big, uint32_t (&lo)[2], uint32_t (&hi)[2]) {
#pragma unroll
    for (int i = 0; i < 2; i++) {  // 1024 + n, 1024 + 16 n
        const half2v l = as_half2((w >> (8 * i) & 0x000f000fu) | big), h = as_half2((w >> (8 * i) & 0x00f000f0u) | big);
        lo[i] = __builtin_bit_cast(uint32_t, l - (half_t)1032);
        hi[i] = __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(h, half2v{(half_t)0.0625, (half_t)0.0625},
                                                                       half2v{(half_t)-72, (half_t)-72}));
    }
}
TSL_DEV half8 half8_of(uint32_t a, uint32_t b, uint32_t c, uint32_t d) { return __builtin_bit_cast(half8, u32x4{a, b, c, d}); }

TSL_DEV float lo_h(uint32_t w) { return (float)as_half2(w)[0]; }
TSL_DEV float hi_h(uint32_t w) { return (float)as_half2(w)[1]; }

// The value of the lane that holds token T in this lane's row of 16 (row_newbcast).
TSL_DEV uint32_t of_token(uint32_t x, int t) {
    switch (t) {
#define Q4_TOKEN(T) \
    case T: return __builtin_amdgcn_mov_dpp((int)x, 0x150 + T, 0xf, 0xf, false);
        Q4_TOKEN(0) Q4_TOKEN(1) Q4_TOKEN(2) Q4_TOKEN(3) Q4_TOKEN(4) Q4_TOKEN(5) Q4_TOKEN(6) Q4_TOKEN(7)
        Q4_TOKEN(8) Q4_TOKEN(9) Q4_TOKEN(10) Q4_TOKEN(11) Q4_TOKEN(12) Q4_TOKEN(13) Q4_TOKEN(14)
#undef Q4_TOKEN
        default: return __builtin_amdgcn_mov_dpp((int)x, 0x15f, 0xf, 0xf, false);
    }
}

// (low, step) pairs of a lane's tokens: CF = 1 holds one token's a lane and
// hands them round, else a lane loads its own 16 / CF.
template <int CF>
struct Pairs {
    Words<4> w[4 / CF];
    TSL_DEV void load(const u16* p, long block, int l16) {
        const uint8_t* q = reinterpret_cast<const uint8_t*>(p + block * 32) + (l16 / (16 / CF)) * (64 / CF);
#pragma unroll
        for (int i = 0; i < 4 / CF; i++) w[i].load(q + 16 * i);
    }
    TSL_DEV uint32_t get(int i) const { return w[i / 4].w[i % 4]; }
    TSL_DEV uint32_t most() const {  // the largest step's bits (in the upper half)
        uint32_t x = 0;
#pragma unroll
        for (int i = 0; i < 16 / CF; i++) x = max(x, w[i / 4].w[i % 4] & 0x7fff0000u);
        return x;
    }
    TSL_DEV void drop(int first, int left, bool all) {  // tokens first + .. at left and past it, or all of them
#pragma unroll
        for (int i = 0; i < 16 / CF; i++)
            if (all || first + i >= left) w[i / 4].w[i % 4] = 0;
    }
};
template <>
struct Pairs<1> {
    uint32_t w;
    TSL_DEV void load(const u16* p, long block, int l16) { w = reinterpret_cast<const uint32_t*>(p)[block * 16 + l16]; }
    TSL_DEV uint32_t get(int i) const { return of_token(w, i); }
    TSL_DEV uint32_t most() const { return w & 0x7fff0000u; }
    TSL_DEV void drop(int, int left, bool all) {
        if (all || (int)(threadIdx.x & 15) >= left) w = 0;
    }
};

template <int D, int CF>
struct Q4Tile {
    Words<D / 32> k[4];  // tile i: token 4 i + l % 4 of block (l % 16) / 4, bytes (D / 8) (l / 16) ..
    Words<4> v[D / 32];  // channel pair 16 j + l % 16, the 16 tokens of block l / 16
    Pairs<CF> ks, vs;    // of this lane's tokens of block l / 16
};

// Lanes 16 / CF j .. of every row of 16 take part j's value from the row's first lanes (pack), and back (part).
template <int CF>
TSL_DEV float pack_lanes(const float (&s)[CF]) {
    int v = __builtin_bit_cast(int, s[0]);
    if constexpr (CF == 2) {
        v = __builtin_amdgcn_update_dpp(v, __builtin_bit_cast(int, s[1]), 0x118, 0xf, 0xc, false);  // row_shr:8
    } else if constexpr (CF == 4) {
        v = __builtin_amdgcn_update_dpp(v, __builtin_bit_cast(int, s[1]), 0x114, 0xf, 0x2, false);  // row_shr:4, 8, 12
        v = __builtin_amdgcn_update_dpp(v, __builtin_bit_cast(int, s[2]), 0x118, 0xf, 0x4, false);
        v = __builtin_amdgcn_update_dpp(v, __builtin_bit_cast(int, s[3]), 0x11c, 0xf, 0x8, false);
    }
    return __builtin_bit_cast(float, v);
}
template <int CF>
TSL_DEV uint32_t part_lanes(uint32_t x, int j) {
    if (j == 0) return x;
    if constexpr (CF == 2) return __builtin_amdgcn_mov_dpp((int)x, 0x108, 0xf, 0xf, true);  // row_shl:8
    if (j == 1) return __builtin_amdgcn_mov_dpp((int)x, 0x104, 0xf, 0xf, true);
    if (j == 2) return __builtin_amdgcn_mov_dpp((int)x, 0x108, 0xf, 0xf, true);
    return __builtin_amdgcn_mov_dpp((int)x, 0x10c, 0xf, 0xf, true);
}
// Over the lanes that share a head: those 16 / CF apart in a row, and the four rows.
template <int CF>
TSL_DEV float head_max(float x) {
    if constexpr (CF >= 2) x = fmaxf(x, __shfl_xor(x, 8));
    if constexpr (CF >= 4) x = fmaxf(x, __shfl_xor(x, 4));
    x = fmaxf(x, xor16(x));
    return fmaxf(x, xor32(x));
}
template <int CF>
TSL_DEV float head_sum(float x) {
    if constexpr (CF >= 2) x += __shfl_xor(x, 8);
    if constexpr (CF >= 4) x += __shfl_xor(x, 4);
    x += xor16(x);
    return x + xor32(x);
}

// The sequence of slot s by length: slots 0 .. first - 1 the longest ones, longest first, the others the rest, shortest
// first (of equal ones the first sequence is the longest). Every wavefront by itself: the r-th largest length bit by
// bit, by counting the lengths at or above each candidate.
TSL_DEV int by_length(const Q4Args& a, int s) {
    constexpr int NV = RANKED / 64;
    const int lane = threadIdx.x & 63;
    const int r = s < a.first ? s : a.B - 1 - (s - a.first);
    int v[NV];
#pragma unroll
    for (int i = 0; i < NV; i++) {
        v[i] = -1;
        if (64 * i < a.B && 64 * i + lane < a.B) v[i] = tokens_of(a, 64 * i + lane);
    }
    auto count = [&](int least) {
        int n = 0;
#pragma unroll
        for (int i = 0; i < NV; i++)
            if (64 * i < a.B) n += __popcll(__builtin_amdgcn_ballot_w64(v[i] >= least));
        return n;
    };
    int at = 0;
    for (int bit = 31 - __builtin_clz((unsigned)(a.MP * a.P)); bit >= 0; bit--)
        if (count(at | 1 << bit) > r) at |= 1 << bit;
    int k = r - count(at + 1), b = 0;  // the k-th of those of this length
#pragma unroll
    for (int i = 0; i < NV; i++) {
        if (64 * i >= a.B) break;
        const uint64_t same = __builtin_amdgcn_ballot_w64(v[i] == at);
        const int before = __builtin_amdgcn_mbcnt_hi((uint32_t)(same >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)same, 0));
        const uint64_t hit = __builtin_amdgcn_ballot_w64(v[i] == at && before == k);
        if (hit) b = 64 * i + __builtin_ctzll(hit);
        k -= __popcll(same);
    }
    return b;
}

template <int D, int QPG, int NW>
__global__ __launch_bounds__(64 * NW, D == 128 || NW == 8 ? 2 : 3) void decode_q4_mfma(Q4Args a) {
    constexpr int KW = D / 32, NT = D / 16, CB = D / 8;  // words of a K row a lane; channel tiles; their bytes
    // p = 2^(cs (u - m) + lift): m a maximum of u that may grow by 2^GROW before it is moved, lift such that p step
    // stays below 2^15 for the largest step met: small values keep their f16 bits too.
    constexpr float GROW = 2.0f;
    // Few query heads leave most of the 16 columns empty: the scores of four (two)
    // of a lane's tiles are packed onto the row's lanes, 16 / CF a lane, for the softmax.
    constexpr int CF = QPG <= 4 ? 4 : QPG == 8 ? 2 : 1, TPL = 16 / CF;
    constexpr int COLS = D + 2;
    __shared__ float red[NW][QPG][COLS];
    __shared__ int tab[CHUNK_MAX / 16];
    TSL_POISON(red); TSL_POISON(tab);
    const int lane = threadIdx.x & 63, l16 = lane & 15, g4 = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // Chunk after chunk: workgroups go round the XCDs, and with a sequence's chunks side by side some XCDs had
    // the first ones, which all sequences have, and others the last (64 of 128-4096 tokens 57.7 us).
    const int c = blockIdx.x / (a.B * a.G), slot = blockIdx.x % (a.B * a.G);
    const int g = slot % a.G, b = NW == 4 && a.first ? by_length(a, slot / a.G) : slot / a.G, bg = b * a.G + g;
    // The length, the chunk's table entries (t_in: where in its first page it begins) and q in
    // one round trip: none of these loads depends on another.
    const int t_lo = c * a.CT, t_in = t_lo & (a.P - 1);
    const int held = (t_in + min(a.CT, a.MP * a.P - t_lo) + a.P - 1) >> a.pshift;
    for (int e = threadIdx.x; e < held; e += 64 * NW) tab[e] = a.table[(long)b * a.MP + (t_lo >> a.pshift) + e];
    float qs[2 * CB];
#pragma unroll
    for (int i = 0; i < 2 * CB; i++) qs[i] = 0.0f;
    if (l16 < QPG) {  // head l16's channels 2 CB g4 .. 2 CB g4 + 2 CB - 1
        const u16* qp = a.Q + ((long)b * a.H + g * QPG + l16) * D + 2 * CB * g4;
#pragma unroll
        for (int i = 0; i < CB / 4; i++) {
            const u32x4 t = *reinterpret_cast<const u32x4u*>(qp + 8 * i);
#pragma unroll
            for (int e = 0; e < 8; e++) qs[8 * i + e] = h2f((u16)(t[e >> 1] >> (16 * (e & 1))));
        }
    }
    const int n = tokens_of(a, b);
    const int len = min(n - t_lo, a.CT);  // this chunk's tokens
    if (len <= 0) {
        if (c == 0)  // an empty sequence: 0 / 0
            for (int i = threadIdx.x; i < QPG * D; i += 64 * NW) a.O[((long)b * a.H + g * QPG) * D + i] = 0x7e00;
        return;
    }
    const int entries = (t_in + len + a.P - 1) >> a.pshift;
    __syncthreads();  // (tab)

    // Word w's eight channels are a step's operand.
    float qmax = 0.0f, qsum = 0.0f;
#pragma unroll
    for (int i = 0; i < 2 * CB; i++) {
        qmax = fmaxf(qmax, __builtin_fabsf(qs[i]));
        qsum += qs[i];
    }
    qmax = fmaxf(qmax, xor16(qmax));
    qmax = fmaxf(qmax, xor32(qmax));
    qsum += xor16(qsum);
    qsum += xor32(qsum);
    // 2^eq brings the largest magnitude into [2^10, 2^11); an infinity or zeros stay.
    const int eq = qmax > 0.0f && qmax <= 65504.0f ? 10 - __builtin_amdgcn_frexp_expf(qmax) + 1 : 0;
    const float up = __builtin_ldexpf(a.c2 < 0.0f ? -1.0f : 1.0f, eq);  // (a negative scale: q turned over)
    half8 qop[KW];
#pragma unroll
    for (int w = 0; w < KW; w++) {
        // Nibble e of a word is channel 8 w + e; its operand order: 0 4 2 6 (low) 1 5 3 7 (high).
        constexpr int at[8] = {0, 4, 2, 6, 1, 5, 3, 7};
#pragma unroll
        for (int e = 0; e < 8; e++) qop[w][e] = (half_t)(qs[8 * w + at[e]] * up);
    }
    // Of the head whose scores this lane takes (l16 % TPL): u's units (a scale of 0: nearly), and low's factor.
    const int head = (lane & 48) + l16 % TPL;
    const float unit = __builtin_ldexpf(__builtin_fabsf(a.c2), 18 - eq);
    const float cs = __shfl(unit < 1e-37f ? 1e-37f : unit, head);  // (a NaN stays)
    const float qz = __shfl(__builtin_ldexpf(qsum, eq - 18) * (a.c2 < 0.0f ? -1.0f : 1.0f), head);

    const int ntiles = (len + TILE - 1) / TILE;
    const int kb = (l16 >> 2), kt = l16 & 3;  // this lane's block and token of K's tiles
    const int blocks = a.P >> 4;              // blocks of 16 tokens a page
    // The page of the chunk's p-th block of 16 tokens (-1: outside the pool or past the chunk), and
    // where the block is in the pool (page 0's for none: its bytes are read, its pairs are not used).
    auto page_at = [&](int p) {
        const int e = (t_in + 16 * p) >> a.pshift;
        const int page = tab[min(e, entries - 1)];
        return e < entries && page < a.NP ? page : -1;
    };
    auto block_at = [&](int p) { return ((long)max(page_at(p), 0) * a.G + g) * blocks + (((t_in >> 4) + p) & (blocks - 1)); };
    // Loads are issued whether or not the tile exists (past the chunk the last one's again, from the caches): behind
    // a branch the compiler could not count on them and waited for all.
    auto load = [&](int tile, Q4Tile<D, CF>& x) {
        tile = min(tile, ntiles - 1);
        const long bk = block_at(4 * tile + kb), bv = block_at(4 * tile + g4);
        const uint8_t* kp = a.Kc + bk * (8 * D) + kt * (D / 2) + CB * g4;
#pragma unroll
        for (int i = 0; i < 4; i++) x.k[i].load(kp + i * (2 * D));
        x.ks.load(a.Ks, bv, l16);
        x.vs.load(a.Vs, bv, l16);
        const uint8_t* vp = a.Vc + bv * (8 * D) + l16 * 16;
#pragma unroll
        for (int j = 0; j < KW; j++) x.v[j].load(vp + j * 256);
    };

    float m = -INFINITY, l = 0.0f, low = 0.0f;  // maximum of u; sums of p and p (low + 8 step) (this lane's tokens)
    float lift = 0.0f;                         // (these two of the wavefront)
    uint32_t most = 0;                         // steps below this bound need no other lift
    uint32_t big = 0x64006400u;
    asm("" : "+v"(big));
    float4v acc[NT];
#pragma unroll
    for (int i = 0; i < NT; i++) acc[i] = float4v{};
    auto step = [&](int tile, Q4Tile<D, CF>& x) {
        // Tokens past the end, and pages outside the pool: pairs of zeros (what the
        // cache holds there is not looked at; a spoilt pair would spoil 0 x it).
        const int left = len - tile * TILE - 16 * g4;  // of this lane's block
        const int first = (l16 / TPL) * (CF == 1 ? 0 : TPL);  // this lane's tokens of it: first ..
        const bool none = page_at(4 * tile + g4) < 0, tail = __builtin_amdgcn_ballot_w64(left < 16) != 0;
        if (tail || __builtin_amdgcn_ballot_w64(none)) {
            x.ks.drop(first, left, none);
            x.vs.drop(first, left, none);
        }
        float4v s[4];
#pragma unroll
        for (int t = 0; t < 4; t++) {
            s[t] = float4v{};
#pragma unroll
            for (int w = 0; w < KW; w++) {
                uint32_t nl[2], nh[2];
                nibbles(x.k[t].w[w], nl, nh);
                s[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(half8_of(nl[0], nl[1], nh[0], nh[1]), qop[w], s[t], 0, 0, 0);
            }
        }
        float u[TPL];  // token first + i
#pragma unroll
        for (int i = 0; i < TPL; i++) {
            float part[CF];
#pragma unroll
            for (int j = 0; j < CF; j++) part[j] = s[j * (4 / CF) + i / 4][i % 4];
            const uint32_t pair = x.ks.get(i);
            u[i] = __builtin_fmaf(hi_h(pair), pack_lanes<CF>(part), lo_h(pair) * qz);
        }
        if (tail) {
#pragma unroll
            for (int i = 0; i < TPL; i++)
                if (first + i >= left) u[i] = -INFINITY;
        }
        float mx = u[0];
#pragma unroll
        for (int i = 1; i < TPL; i++) mx = fmaxf(mx, u[i]);
        // Some head's maximum moves, or a step passes the bound: all lanes of the heads together.
        const uint32_t sm = x.vs.most();
        if (__builtin_amdgcn_ballot_w64((mx - m) * cs > GROW || sm >= most)) {
            mx = fmaxf(head_max<CF>(mx), m);
            float by = m == mx ? 0.0f : (m - mx) * cs;
            m = mx;
            const float step = wave_max(h2f((u16)(sm >> 16)));  // (NaN and infinite steps have no lift of their own)
            if (__builtin_amdgcn_ballot_w64(sm >= most)) {
                const int e = max(min(step > 0.0f && step <= 65504.0f ? __builtin_amdgcn_frexp_expf(step) : -11, 16), -11);
                const float to = 13.0f - e;  // 2^(lift + GROW + e) = 2^15
                by += to - lift;
                lift = to;
                most = e < 16 ? (uint32_t)(e + 15) << 26 : 0x7c000000u;  // 2^e as f16 bits, in the upper half
            }
            const float f = __builtin_amdgcn_exp2f(by);
            l *= f;
            low *= f;
#pragma unroll
            for (int i = 0; i < NT; i++) acc[i] *= f;
        }
        const float off = lift - m * cs;
        uint32_t ph[8], pl[8];  // p step in two f16, in V's token order: 0 2, 1 3 of every four
#pragma unroll
        for (int t = 0; t < TPL / 4; t++) {
            half_t h[4], e[4];
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(u[4 * t + r], cs, off));
                const uint32_t pair = x.vs.get(4 * t + r);
                l += p;
                low = __builtin_fmaf(p, __builtin_fmaf(8.0f, hi_h(pair), lo_h(pair)), low);
                float w = p * hi_h(pair);
                asm("" : "+v"(w));  // (both halves of one f32 value: else one comes of the product rounded to f16 at once)
                h[r] = (half_t)w;
                e[r] = (half_t)(w - (float)h[r]);
            }
            const uint32_t h0 = __builtin_bit_cast(uint32_t, half2v{h[0], h[2]}), h1 = __builtin_bit_cast(uint32_t, half2v{h[1], h[3]});
            const uint32_t e0 = __builtin_bit_cast(uint32_t, half2v{e[0], e[2]}), e1 = __builtin_bit_cast(uint32_t, half2v{e[1], e[3]});
#pragma unroll
            for (int j = 0; j < CF; j++) {
                const int at = 2 * (j * (4 / CF) + t);
                ph[at] = part_lanes<CF>(h0, j), ph[at + 1] = part_lanes<CF>(h1, j);
                pl[at] = part_lanes<CF>(e0, j), pl[at + 1] = part_lanes<CF>(e1, j);
            }
        }
#pragma unroll
        for (int s = 0; s < 2; s++) {
            const half8 hp = half8_of(ph[4 * s], ph[4 * s + 1], ph[4 * s + 2], ph[4 * s + 3]);
            const half8 ep = half8_of(pl[4 * s], pl[4 * s + 1], pl[4 * s + 2], pl[4 * s + 3]);
#pragma unroll
            for (int j = 0; j < D / 32; j++) {
                uint32_t l0[2], h0[2], l1[2], h1[2];
                centred(x.v[j].w[2 * s], big, l0, h0);
                centred(x.v[j].w[2 * s + 1], big, l1, h1);
                const half8 even = half8_of(l0[0], l0[1], l1[0], l1[1]), odd = half8_of(h0[0], h0[1], h1[0], h1[1]);
                acc[2 * j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(even, hp, acc[2 * j], 0, 0, 0);
                acc[2 * j + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(odd, hp, acc[2 * j + 1], 0, 0, 0);
                acc[2 * j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(even, ep, acc[2 * j], 0, 0, 0);
                acc[2 * j + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(odd, ep, acc[2 * j + 1], 0, 0, 0);
            }
        }
    };
    Q4Tile<D, CF> x, y;
    load(wave, x);
    for (int t = wave; t < ntiles; t += 2 * NW) {
        load(t + NW, y);
        step(t, x);
        if (t + NW >= ntiles) break;
        load(t + 2 * NW, x);
        step(t + NW, y);
    }
    // The wavefronts' states, joined in order: the maximum (log2 units), sums, outputs.
    l = head_sum<CF>(l);
    low = head_sum<CF>(low);
    if (l16 < QPG) {
#pragma unroll
        for (int j = 0; j < D / 32; j++)
#pragma unroll
            for (int e = 0; e < 2; e++)
#pragma unroll
                for (int r = 0; r < 4; r++)
                    red[wave][l16][2 * (16 * j + 4 * g4 + r) + e] = acc[2 * j + e][r] + low;
        if (g4 == 0) red[wave][l16][D] = m * cs - lift, red[wave][l16][D + 1] = l;
    }
    __syncthreads();
    const int active = min(NW, ntiles);
    for (int i = threadIdx.x; i < QPG * D; i += 64 * NW) {
        const int h = i / D, d = i % D;
        float top = red[0][h][D];
        for (int w = 1; w < active; w++) top = fmaxf(top, red[w][h][D]);
        float sum = 0.0f, v = 0.0f;
        for (int w = 0; w < active; w++) {
            const float f = __builtin_amdgcn_exp2f(red[w][h][D] - top);
            sum = __builtin_fmaf(red[w][h][D + 1], f, sum);
            v = __builtin_fmaf(red[w][h][d], f, v);
        }
        if (a.NCH == 1) {
            a.O[((long)b * a.H + g * QPG + h) * D + d] = f2h(v / sum);
        } else {
            float* p = a.part + (((long)bg * a.NCH + c) * QPG + h) * (2 + D);
            if (d == 0) p[0] = top, p[1] = sum;
            p[2 + d] = v;
        }
    }
}

// Joins a (sequence, query head)'s chunks in order. Four wavefronts take every fourth chunk.
template <int D>
__global__ __launch_bounds__(256) void decode_q4_join(Q4Args a, int qpg) {
    __shared__ float red[4][D + 2];
    TSL_POISON(red);
    const int h = blockIdx.x % a.H, g = h / qpg, i = h % qpg;
    const long b = blockIdx.x / a.H;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int nact = (int)(((long)tokens_of(a, b) + a.CT - 1) / a.CT);
    if (nact == 0) return;  // (an empty sequence: written already)
    const float* p = a.part + ((b * a.G + g) * a.NCH * qpg + i) * (2L + D);
    const long next = (long)qpg * (2 + D);
    float m = -INFINITY, l = 0.0f, v[(D + 63) / 64];
    for (int c = lane; c < nact; c += 64) m = fmaxf(m, p[c * next]);
    m = wave_max(m);
#pragma unroll
    for (int k = 0; k < (D + 63) / 64; k++) v[k] = 0.0f;
#pragma unroll 4
    for (int c = wave; c < nact; c += 4) {
        const float f = __builtin_amdgcn_exp2f(p[c * next] - m);
        l = __builtin_fmaf(p[c * next + 1], f, l);
#pragma unroll
        for (int k = 0; k < (D + 63) / 64; k++)
            if (D >= 64 || lane < D) v[k] = __builtin_fmaf(p[c * next + 2 + 64 * k + lane], f, v[k]);
    }
#pragma unroll
    for (int k = 0; k < (D + 63) / 64; k++)
        if (D >= 64 || lane < D) red[wave][64 * k + lane] = v[k];
    if (lane == 0) red[wave][D] = l;
    __syncthreads();
    if (threadIdx.x < D) {
        const int d = threadIdx.x;
        const float sum = (red[0][D] + red[1][D]) + (red[2][D] + red[3][D]);
        a.O[(b * a.H + h) * D + d] = f2h(((red[0][d] + red[1][d]) + (red[2][d] + red[3][d])) / sum);
    }
}

// Tokens a chunk: about two workgroups of 4 wavefronts a CU at the table's full length, which run at one time;
// 512 at least. A workgroup costs 4 us of latencies before and after its tiles, and a second chunk the
// join, 5 us (sequences in order): 64 x 128-4096 tokens, 8 kv heads of 128, chunks of 512 / 1024 / 2048 / 4096 55 / 45 / 45 / 39 us, all
// 4096 82 / 63 / 57 / 52; one sequence of 16384 11.3 / 13.2 / 18.4 / 28.1, 16 x 100-4000 22.2 /
// 18.8 / 19.4 / 24.9. Tables of at most ONE_CHUNK tokens are one chunk of 8 wavefronts
// (5 x 20-333 tokens, 4 kv heads of 64, 5.8 us, 4 wavefronts 6.5).
constexpr int ONE_CHUNK = 1024;
int chunk_tokens(const TslKernel& k) {
    const int64_t bg = std::max<int64_t>(1, k.dim("B") * k.dim("G")), most = k.dim("MP") * k.dim("P");
    if (most <= ONE_CHUNK) return ONE_CHUNK;
    return (int)std::min<int64_t>(std::max<int64_t>(512, (most * bg / (2 * num_cus()) + 255) / 256 * 256), CHUNK_MAX);
}
int nchunks(const TslKernel& k) {
    const int64_t most = k.dim("MP") * k.dim("P"), ct = chunk_tokens(k);
    return (int)std::max<int64_t>(1, (most + ct - 1) / ct);
}

// Sequences by length (by_length), where a CU has more than one workgroup, at most two, tables are long and of two chunks
// at most: the one that comes second to a CU is short where the first is long. us, in order / by length: 64 x 128-4096
// tokens, 8 kv heads of 128, 39.5 / 32.9, 48 of them 37.0 / 32.3, 34 30.2 / 29.3, 120 x 100-4000, 4 of 64, 35.9 / 30.3; the
// price, one more round trip, where all have 4096 52.0 / 52.9 (by longest first for 1600 workgroups 12 % more, for
// tables of 16000 tokens, 4 chunks, 2 %: left in order).
int ranked_first(const TslKernel& k) {
    const int64_t B = k.dim("B"), G = k.dim("G"), cus = num_cus();
    if (k.dim("MP") * k.dim("P") <= ONE_CHUNK || nchunks(k) > 2 || B * G <= cus || B * G > 2 * cus || B > RANKED) return 0;
    return (int)((cus + G - 1) / G);
}

template <int D, int QPG>
int run_q4(const Q4Args& a, hipStream_t s) {
    const dim3 grid((unsigned)((long)a.B * a.G * a.NCH));
    if constexpr (D == 16) {
        hipLaunchKernelGGL((decode_q4_any<D, QPG>), grid, dim3(256), 0, s, a);
    } else {
        if (a.wide) hipLaunchKernelGGL((decode_q4_mfma<D, QPG, 8>), grid, dim3(512), 0, s, a);
        else hipLaunchKernelGGL((decode_q4_mfma<D, QPG, 4>), grid, dim3(256), 0, s, a);
    }
    int r = TSL_LAUNCHED("quant decode_attention");
    if (r || a.NCH == 1) return r;
    hipLaunchKernelGGL(decode_q4_join<D>, dim3((unsigned)((long)a.B * a.H)), dim3(256), 0, s, a, QPG);
    return TSL_LAUNCHED("quant decode_attention join");
}

template <int D>
int run_q4_d(const Q4Args& a, hipStream_t s) {
    switch (a.H / a.G) {
        case 1: return run_q4<D, 1>(a, s);
        case 2: return run_q4<D, 2>(a, s);
        case 4: return run_q4<D, 4>(a, s);
        case 8: return run_q4<D, 8>(a, s);
        default: return run_q4<D, 16>(a, s);
    }
}

}  // namespace

int setup_decode_q4(TslKernel& k) {
    if (int r = check_cache_q4(k)) return r;
    const int64_t H = k.dim("H"), G = k.dim("G"), B = k.dim("B"), MP = k.dim("MP");
    if (H % G != 0) return tsl_fail(-2, "quant/decode_attention: H must be a multiple of G");
    const int64_t qpg = H / G;
    if (qpg != 1 && qpg != 2 && qpg != 4 && qpg != 8 && qpg != 16)
        return tsl_fail(-2, "quant/decode_attention: H / G must be 1, 2, 4, 8 or 16");
    if (k.dim("NP") == 0) return tsl_fail(-2, "quant/decode_attention: a pool of no pages");
    // (a launch holds less than 2^32 work-items, 512 at most for each of these)
    if (MP > INT_MAX / k.dim("P") || B > (1 << 22) || H > (1 << 22) || B * H > (1 << 22) || B * G * nchunks(k) > (1 << 22))
        return tsl_fail(-2, "quant/decode_attention: at most 2^31 - 1 tokens a table and 2^22 (sequence, head, chunk)s");
    return nchunks(k) > 1 ? tsl_scratch(k, (size_t)B * H * nchunks(k) * (2 + k.dim("D")) * sizeof(float)) : 0;
}

int launch_decode_q4(TslKernel& k, const uint64_t* args, hipStream_t s) {
    Q4Args a{};
    a.Q = P<u16>(args[0]);
    a.Kc = P<uint8_t>(args[1]);
    a.Vc = P<uint8_t>(args[2]);
    a.Ks = P<u16>(args[3]);
    a.Vs = P<u16>(args[4]);
    a.table = P<int>(args[5]);
    a.lens = P<int>(args[6]);
    a.O = P<u16>(args[7]);
    a.c2 = arg_f32(args[8]) * LOG2E;
    a.B = k.dim("B"), a.H = k.dim("H"), a.G = k.dim("G"), a.NP = k.dim("NP"), a.P = k.dim("P"), a.MP = k.dim("MP");
    a.NCH = nchunks(k), a.CT = chunk_tokens(k), a.pshift = __builtin_ctz((unsigned)a.P);
    a.wide = (int64_t)a.MP * a.P <= ONE_CHUNK;
    a.first = ranked_first(k);
    a.part = reinterpret_cast<float*>(k.scratch);
    if (a.B == 0) return 0;
    // (slices of a pool by layer or page are aligned so: 16 tokens' codes are 128 bytes at least)
    if ((args[1] | args[2]) % 16 || (args[3] | args[4]) % 16)
        return tsl_fail(-2, "quant/decode_attention: Kc, Vc, Ks and Vs must be 16-byte aligned");
    switch (k.dim("D")) {
        case 16: return run_q4_d<16>(a, s);
        case 32: return run_q4_d<32>(a, s);
        case 64: return run_q4_d<64>(a, s);
        default: return run_q4_d<128>(a, s);
    }
}
