// Rows in 8 bits and the 4-bit cache's write (the `quant` kernels; not .tl
// kernels): quantize, rmsnorm and add_rmsnorm with 8-bit outputs, kv_write.
//
// 8 bits: a row y has the step s = max |y| / 127 and the codes q = the whole
// number nearest to y / s, an even one on a tie. 4 bits: a head's vector x of
// one token has the lowest value lo, the step (hi - lo) / 15 rounded to f16,
// and the codes nearest to 15 (x - lo) / (hi - lo). Every code is the
// correctly rounded one: a quotient is first taken with a rounded
// reciprocal, and where it lies so near a border that its error could decide,
// the two sides of the tie are compared as products of a few bits, which are
// exact. So codes do not depend on how rows are spread over threads.
//
// A row or head that holds a NaN or an infinity has the scale (pair) NaN and codes 0:
// whatever is computed from it is NaN.
#include "common.h"

#include <algorithm>
#include <climits>
#include <type_traits>

namespace {

typedef u32x4 u32x4u __attribute__((aligned(2)));
typedef float4v float4u __attribute__((aligned(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef u32x2 u32x2u __attribute__((aligned(1)));
typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32u __attribute__((aligned(2)));

TSL_DEV u32x4 load8(const u16* p) { return *reinterpret_cast<const u32x4u*>(p); }
TSL_DEV float4v load4(const float* p) { return *reinterpret_cast<const float4u*>(p); }
TSL_DEV u16 half_of(const u32x4& v, int i) { return (u16)(v[i >> 1] >> (16 * (i & 1))); }

// Doubles across a wavefront, as wave_max / wave_sum (common.h) do floats.
template <int CTRL>
TSL_DEV double dpp64(double x) {
    const uint64_t b = __builtin_bit_cast(uint64_t, x);
    const uint32_t lo = __builtin_amdgcn_mov_dpp((int)(uint32_t)b, CTRL, 0xf, 0xf, false);
    const uint32_t hi = __builtin_amdgcn_mov_dpp((int)(uint32_t)(b >> 32), CTRL, 0xf, 0xf, false);
    return __builtin_bit_cast(double, ((uint64_t)hi << 32) | lo);
}
TSL_DEV double lane_value64(double x, int lane) {
    const uint64_t b = __builtin_bit_cast(uint64_t, x);
    const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)b, lane);
    const uint32_t hi = __builtin_amdgcn_readlane((int)(uint32_t)(b >> 32), lane);
    return __builtin_bit_cast(double, ((uint64_t)hi << 32) | lo);
}
TSL_DEV double wave_max64(double x) {
    x = fmax(x, dpp64<DPP_XOR1>(x));
    x = fmax(x, dpp64<DPP_XOR2>(x));
    x = fmax(x, dpp64<DPP_HALF_MIRROR>(x));
    x = fmax(x, dpp64<DPP_MIRROR>(x));
    return fmax(fmax(lane_value64(x, 0), lane_value64(x, 16)), fmax(lane_value64(x, 32), lane_value64(x, 48)));
}
TSL_DEV double wave_sum64(double x) {
    x += dpp64<DPP_XOR1>(x);
    x += dpp64<DPP_XOR2>(x);
    x += dpp64<DPP_HALF_MIRROR>(x);
    x += dpp64<DPP_MIRROR>(x);
    return (lane_value64(x, 0) + lane_value64(x, 16)) + (lane_value64(x, 32) + lane_value64(x, 48));
}

// Codes of values p in a row whose largest magnitude is top > 0: t = 127 p / top from
// inv = 127 / top, rounded to a whole number by adding 1.5 2^23 (f32; 1.5 2^52 f64), which leaves
// the code in the sum's low byte. NEAR is above t's error (127 x 2 half-steps of the type);
// closer to a tie than that, 254 |p| is compared with (2 k + 1) top: p and top
// of 11 bits (f16) give 19-bit products, exact in f32; products of f32 and f16 (35 bits) give 43-bit
// ones, exact in f64. One test for 8 values: with one for each, 4096 x 5632 took 15.9 us, 14.0 so (69 MB; the
// card copies 67 MB in that).
template <class F>
struct Code8 {
    static constexpr bool WIDE = sizeof(F) == 8;
    static constexpr F MAGIC = WIDE ? (F)6755399441055744.0 : (F)12582912.0, NEAR = WIDE ? (F)1e-12 : (F)5e-5;
    F top, inv;
    TSL_DEV explicit Code8(F t) : top(t), inv(t > 0 ? (F)127 / t : (F)0) {}
    TSL_DEV int exact(F p) const {
        const F t = p * inv, n = __builtin_elementwise_roundeven(t), a = __builtin_elementwise_abs(p);
        if (__builtin_elementwise_abs(t - n) <= (F)0.5 - NEAR) return (int)n;
        const F k = __builtin_elementwise_floor(__builtin_elementwise_abs(t)), l = (F)254 * a, r = ((F)2 * k + 1) * top;
        const int m = (int)k + (l > r || (l == r && ((int)k & 1)));
        return p < 0 ? -m : m;
    }
    TSL_DEV u32x2 operator()(const F (&p)[8]) const {  // eight codes as bytes
        u32x2 v;
        F off = 0;
#pragma unroll
        for (int h = 0; h < 2; h++) {
            uint32_t c[4];
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const F u = __builtin_elementwise_fma(p[4 * h + e], inv, MAGIC), n = u - MAGIC;
                off = __builtin_elementwise_max(off, __builtin_elementwise_abs(__builtin_elementwise_fma(p[4 * h + e], inv, -n)));
                if constexpr (WIDE) c[e] = (uint32_t)__builtin_bit_cast(uint64_t, u) & 255;
                else c[e] = __builtin_bit_cast(uint32_t, u) & 255;
            }
            v[h] = c[0] | c[1] << 8 | c[2] << 16 | c[3] << 24;
        }
        if (off > (F)0.5 - NEAR)
#pragma unroll
            for (int h = 0; h < 2; h++)
                v[h] = (uint32_t)(exact(p[4 * h]) & 255) | (uint32_t)(exact(p[4 * h + 1]) & 255) << 8 |
                       (uint32_t)(exact(p[4 * h + 2]) & 255) << 16 | (uint32_t)exact(p[4 * h + 3]) << 24;
        return v;
    }
};

// Reductions over the NT threads that share a row (NT = 64: a wavefront of
// its own); red: NT / 64 values, free again after the next barrier.
template <int NT, class T, class WaveOp, class Op>
TSL_DEV T row_reduce(T x, T* red, WaveOp wave, Op op) {
    x = wave(x);
    if constexpr (NT == 64) return x;
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = x;
    __syncthreads();
    x = red[0];
#pragma unroll
    for (int w = 1; w < NT / 64; w++) x = op(x, red[w]);
    return x;
}

// 8 codes to row q at column c of K (8-byte stores at any alignment; byte by byte
// where the chunk crosses the row's end).
TSL_DEV void store_codes(int8_t* q, int c, int K, u32x2 v) {
    if (c + 8 <= K) {
        *reinterpret_cast<u32x2u*>(q + c) = v;
    } else {
#pragma unroll
        for (int e = 0; e < 8; e++)
            if (c + e < K) q[c + e] = (int8_t)(v[e >> 2] >> (8 * (e & 3)));
    }
}

// 8 f16 of a row from column c (zeros past K).
TSL_DEV u32x4 row8(const u16* p, int c, int K) {
    if (c + 8 <= K) return load8(p + c);
    u32x4 v = {0, 0, 0, 0};
#pragma unroll
    for (int e = 0; e < 8; e++)
        if (c + e < K) v[e >> 1] |= (uint32_t)p[c + e] << (16 * (e & 1));
    return v;
}
TSL_DEV void row8f(const float* p, int c, int K, float (&r)[8]) {
    if (c + 8 <= K) {
        const float4v a = load4(p + c), b = load4(p + c + 4);
#pragma unroll
        for (int e = 0; e < 4; e++) r[e] = a[e], r[4 + e] = b[e];
    } else {
#pragma unroll
        for (int e = 0; e < 8; e++) r[e] = c + e < K ? p[c + e] : 0.0f;
    }
}

// quantize: X f16 [M, K] -> Q i8 [M, K], S f32 [M]. NT threads a row, CH
// chunks of 8 columns each held in registers (CH = 0: rows of any length,
// read twice). Magnitudes are compared as their 15 bits, two at a time;
// infinities and NaNs are the largest of them (0x7c00 and up).
template <int NT, int CH>
__global__ __launch_bounds__(NT < 256 ? 256 : NT) void quantize_kernel(const u16* __restrict__ X, int8_t* __restrict__ Q,
                                                                      float* __restrict__ S, int M, int K) {
    constexpr int RPB = NT < 256 ? 256 / NT : 1;
    __shared__ float red[RPB * (NT / 64)];
    TSL_POISON(red);
    const int t = threadIdx.x % NT;
    auto top_of = [](const u32x4& v, u16x2& m) {
#pragma unroll
        for (int i = 0; i < 4; i++)
            m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, (uint32_t)(v[i] & 0x7fff7fffu)));
    };
    for (long row = (long)blockIdx.x * RPB + threadIdx.x / NT; row < M; row += (long)gridDim.x * RPB) {
        const u16* x = X + row * K;
        u32x4 v[CH ? CH : 1];
        u16x2 m = {0, 0};
        if constexpr (CH > 0) {
#pragma unroll
            for (int c = 0; c < CH; c++) v[c] = row8(x, 8 * (c * NT + t), K);
#pragma unroll
            for (int c = 0; c < CH; c++) top_of(v[c], m);
        } else {
            for (int c = 8 * t; c < K; c += 8 * NT) top_of(row8(x, c, K), m);
        }
        const float bits = row_reduce<NT>((float)max(m[0], m[1]), red, wave_max, fmaxf);
        const bool bad = bits >= (float)0x7c00;
        const float top = bad ? 0.0f : h2f((u16)bits);
        const Code8<float> code(top);
        auto emit = [&](int c, const u32x4& w) {
            float p[8];
#pragma unroll
            for (int e = 0; e < 8; e++) p[e] = h2f(half_of(w, e));
            if (c < K) store_codes(Q + row * K, c, K, bad ? u32x2{0, 0} : code(p));
        };
        if constexpr (CH > 0) {
#pragma unroll
            for (int c = 0; c < CH; c++) emit(8 * (c * NT + t), v[c]);
        } else {
            for (int c = 8 * t; c < K; c += 8 * NT) emit(c, row8(x, c, K));
        }
        if (t == 0) S[row] = bad ? __builtin_nanf("") : top / 127.0f;
        if constexpr (NT > 64) __syncthreads();  // (red)
    }
}

// rmsnorm / add_rmsnorm: (ADD: R += X, rounded to f32,) y = R W / sqrt(mean R^2 + eps) in 8
// bits. The norm is a factor of the whole row, so the codes are those of R W, whose
// products f64 holds exactly; it enters the step alone:
//   S = max |R W| / (127 sqrt(mean R^2 + eps)).
// The squares are summed in f64.
template <int NT, int CH, bool ADD>
__global__ __launch_bounds__(NT < 256 ? 256 : NT) void rmsnorm_q8_kernel(const u16* __restrict__ X, float* __restrict__ R,
                                                                        const u16* __restrict__ W, int8_t* __restrict__ Q,
                                                                        float* __restrict__ S, int M, int K, float eps) {
    constexpr int RPB = NT < 256 ? 256 / NT : 1;
    __shared__ double red[2][RPB * (NT / 64)];
    TSL_POISON(red);
    const int t = threadIdx.x % NT;
    for (long row = (long)blockIdx.x * RPB + threadIdx.x / NT; row < M; row += (long)gridDim.x * RPB) {
        float* rp = R + row * K;
        float r[CH ? CH : 1][8];
        u32x4 w[CH ? CH : 1];
        double top = 0.0, sum = 0.0;
        double worst = 0.0;  // 0 x p: NaN where a value is NaN (fmax drops it) or infinite
        auto load = [&](int c, float (&rr)[8], u32x4& ww) {
            row8f(rp, c, K, rr);
            ww = row8(W, c, K);
            if constexpr (ADD) {
                const u32x4 x = row8(X + row * K, c, K);
#pragma unroll
                for (int e = 0; e < 8; e++) rr[e] += h2f(half_of(x, e));
                if (c + 8 <= K) {
                    *reinterpret_cast<float4u*>(rp + c) = float4v{rr[0], rr[1], rr[2], rr[3]};
                    *reinterpret_cast<float4u*>(rp + c + 4) = float4v{rr[4], rr[5], rr[6], rr[7]};
                } else {
#pragma unroll
                    for (int e = 0; e < 8; e++)
                        if (c + e < K) rp[c + e] = rr[e];
                }
            }
        };
        auto stats = [&](const float (&rr)[8], const u32x4& ww) {
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const double a = rr[e], p = a * (double)h2f(half_of(ww, e));
                top = fmax(top, fabs(p));
                sum = fma(a, a, sum);
                worst = fma(0.0, p, worst);
            }
        };
        if constexpr (CH > 0) {
#pragma unroll
            for (int c = 0; c < CH; c++) load(8 * (c * NT + t), r[c], w[c]);
#pragma unroll
            for (int c = 0; c < CH; c++) stats(r[c], w[c]);
        } else {
            for (int c = 8 * t; c < K; c += 8 * NT) {
                load(c, r[0], w[0]);
                stats(r[0], w[0]);
            }
        }
        sum += worst;
        top = row_reduce<NT>(top, red[0], wave_max64, [](double a, double b) { return fmax(a, b); });
        sum = row_reduce<NT>(sum, red[1], wave_sum64, [](double a, double b) { return a + b; });
        const bool bad = __builtin_isnan(sum);
        const Code8<double> code(bad ? 0.0 : top);
        auto emit = [&](int c, const float (&rr)[8], const u32x4& ww) {
            double p[8];
#pragma unroll
            for (int e = 0; e < 8; e++) p[e] = (double)rr[e] * (double)h2f(half_of(ww, e));
            if (c < K) store_codes(Q + row * K, c, K, bad ? u32x2{0, 0} : code(p));
        };
        if constexpr (CH > 0) {
#pragma unroll
            for (int c = 0; c < CH; c++) emit(8 * (c * NT + t), r[c], w[c]);
        } else {
            // (this thread's own stores of R: the same chunks)
            for (int c = 8 * t; c < K; c += 8 * NT) {
                row8f(rp, c, K, r[0]);
                emit(c, r[0], row8(W, c, K));
            }
        }
        if (t == 0) S[row] = bad ? __builtin_nanf("") : (float)(top / (127.0 * sqrt(sum / K + (double)eps)));
        if constexpr (NT > 64) __syncthreads();  // (red)
    }
}

// kv_write: keys rotated at pos, and values, into K and V [T, G, D] in f16 and into the cache in 4 bits.
// The rotation is llm/kv_write's, x1 c - x2 s and x2 c + x1 s: one product rounded to f32, a multiply-add rounded to
// f32, then f16 (rotate; rope_rotate's multiply-add may be rounded to f16 at once).
//
// A workgroup a token, D / 4 lanes a head: lane j holds channels 2j, 2j + 1 and their rotary
// partners D/2 on, which are the bytes j and D/4 + j of the cache's row. Bound by its chain of loads
// (position, slot, rows, tables) for few tokens.
//
// Of rows that name one slot the last is kept. Up to LOOK tokens every workgroup looks through the later rows' slots (T^2 / 2
// loads, one launch); beyond, a table of each slot's last row is made first (a hash table of 2 T to 4 T entries, two launches
// more). us, look / table: 4 kv heads of 64, 4096 tokens 9.2 / 12.0, 6000 12.4 / 13.4, 8192 17.2 / 15.5, 16384 41 / 22.9; 8 of 128,
// 4096 23.5 / 23.2, 8192 44.5 / 37, 16384 97 / 65.
constexpr int LOOK = 6144;

struct KvArgs {
    const u16* QKV;
    const int *pos, *slot;
    const float *Cs, *Sn;
    uint8_t *Kc, *Vc;
    u16 *Ks, *Vs, *K, *V;
    int T, W, NPOS, G, P;
    long NS;
    unsigned long long* last;  // [1 << bits] (slot + 1) << 32 | its last row, 0: empty (null: no table)
    int bits;
};

// A slot's first place in the table, of 2^bits (Fibonacci hashing: neighbouring slots lie far apart).
TSL_DEV uint32_t place_of(int slot, int bits) { return ((uint32_t)slot * 2654435769u) >> (32 - bits); }

__global__ __launch_bounds__(256) void kv_clear_kernel(KvArgs a) {
    u32x4* to = reinterpret_cast<u32x4*>(a.last);
    const long n = 1L << (a.bits - 1);
    for (long i = blockIdx.x * 256L + threadIdx.x; i < n; i += gridDim.x * 256L) to[i] = u32x4{0, 0, 0, 0};
}

// Every row's slot into the table, with the largest row number of each: whatever order they come in, the table holds the
// same for each slot. At most T of its 2 T places or more are taken, so that a free one is always met.
__global__ __launch_bounds__(256) void kv_last_kernel(KvArgs a) {
    const int t = blockIdx.x * 256 + threadIdx.x;
    if (t >= a.T) return;
    const int at = a.slot[t];
    if (at < 0 || at >= a.NS) return;
    const unsigned long long mine = (unsigned long long)(uint32_t)(at + 1u) << 32 | (uint32_t)t;
    const uint32_t mask = (1u << a.bits) - 1;
    for (uint32_t i = place_of(at, a.bits), n = 0; n <= mask; i = (i + 1) & mask, n++) {
        const unsigned long long was = atomicCAS(a.last + i, 0ull, mine);
        if (was == 0) return;
        if (was >> 32 == mine >> 32) {
            atomicMax(a.last + i, mine);
            return;
        }
    }
}

// The last row that names slot `at` (which one does).
TSL_DEV int last_of(const KvArgs& a, int at) {
    const uint32_t mask = (1u << a.bits) - 1, key = at + 1u;
    for (uint32_t i = place_of(at, a.bits), n = 0; n <= mask; i = (i + 1) & mask, n++) {
        const unsigned long long e = a.last[i];
        if ((uint32_t)(e >> 32) == key) return (int)(uint32_t)e;
        if (e == 0) break;
    }
    return -1;
}

TSL_DEV u16 rotate(float a, float c, float b, float s) {  // a c + b s
    float y = __builtin_fmaf(a, c, b * s);
    asm("" : "+v"(y));
    return f2h(y);
}

// TABLE: a.last is made.
template <int D, bool TABLE>
__global__ __launch_bounds__(512) void kv_write_q4_kernel(KvArgs a) {
    constexpr int D2 = D / 2, LPH = D / 4;
    typedef float float2u __attribute__((ext_vector_type(2), aligned(4)));
    const int t = blockIdx.x, nt = blockDim.x;
    const int p = a.pos[t], at = a.slot[t];
    bool keep;
    if constexpr (TABLE) {
        keep = at >= 0 && at < a.NS && last_of(a, at) == t;
    } else {
        // Every thread looks at its share of the later rows, 8 loads at a time (2003 tokens 8.7 us with one).
        bool later = false;
        for (int u = t + 1 + threadIdx.x; u < a.T; u += 8 * nt) {
            int other[8];
#pragma unroll
            for (int i = 0; i < 8; i++) other[i] = u + i * nt < a.T ? a.slot[u + i * nt] : -1;
#pragma unroll
            for (int i = 0; i < 8; i++) later = later || other[i] == at;
        }
        keep = !__syncthreads_or(later) && at >= 0 && at < a.NS;
    }
    const int lane = threadIdx.x % LPH;
    const long page = keep ? at / a.P : 0;
    const int off = keep ? at % a.P : 0;
    // Head h: key h, or value h - G. Every thread goes round as often (the reductions take whole wavefronts).
    for (int h0 = 0; h0 < 2 * a.G; h0 += nt / LPH) {
        const int h = h0 + threadIdx.x / LPH;
        const bool live = h < 2 * a.G, val = h >= a.G;
        const int g = val ? h - a.G : h;
        const u16* x = a.QKV + (long)t * a.W + (a.W - 2L * a.G * D) + (long)(live ? h : 0) * D + 2 * lane;
        const uint32_t xa = *reinterpret_cast<const u32u*>(x), xb = *reinterpret_cast<const u32u*>(x + D2);
        u16 y[4] = {(u16)xa, (u16)(xa >> 16), (u16)xb, (u16)(xb >> 16)};
        if (!val) {
            float2u c = {0.0f, 0.0f}, s = {0.0f, 0.0f};
            if (p >= 0 && p < a.NPOS) {
                c = *reinterpret_cast<const float2u*>(a.Cs + (long)p * D2 + 2 * lane);
                s = *reinterpret_cast<const float2u*>(a.Sn + (long)p * D2 + 2 * lane);
            }
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const float x1 = h2f(y[i]), x2 = h2f(y[2 + i]);
                y[i] = rotate(x1, c[i], x2, -s[i]);
                y[2 + i] = rotate(x2, c[i], x1, s[i]);
            }
        }
        float lo = INFINITY, hi = -INFINITY;
        bool bad = false;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float f = h2f(y[i]);
            bad = bad || (y[i] & 0x7fff) >= 0x7c00;
            lo = fminf(lo, f);
            hi = fmaxf(hi, f);
        }
        if (bad) lo = -INFINITY, hi = INFINITY;
        // Over the head's lanes (LPH = 4 .. 32, aligned).
        auto both = [&](float l, float u) { lo = fminf(lo, l), hi = fmaxf(hi, u); };
        both(dpp<DPP_XOR1>(lo), dpp<DPP_XOR1>(hi));
        both(dpp<DPP_XOR2>(lo), dpp<DPP_XOR2>(hi));
        if constexpr (LPH >= 8) both(dpp<DPP_HALF_MIRROR>(lo), dpp<DPP_HALF_MIRROR>(hi));
        if constexpr (LPH >= 16) both(dpp<DPP_MIRROR>(lo), dpp<DPP_MIRROR>(hi));
        if constexpr (LPH >= 32) both(xor16(lo), xor16(hi));
        bad = __builtin_isinf(lo) || __builtin_isinf(hi);
        // Codes: differences of f16 values are exact in f64 (41 bits), and so are
        // the two sides of a tie, 30 (x - lo) and (2 k + 1) (hi - lo).
        const double range = (double)hi - (double)lo, inv = !bad && range > 0.0 ? 15.0 / range : 0.0;
        int n[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const double d = bad ? 0.0 : (double)h2f(y[i]) - (double)lo, q = d * inv;
            double r = __builtin_rint(q);
            if (fabs(q - r) > 0.5 - 1e-12) {
                const double k = __builtin_floor(q), l = 30.0 * d, u = (2.0 * k + 1.0) * range;
                r = l > u ? k + 1.0 : l < u ? k : 2.0 * __builtin_rint(0.5 * (k + 0.5));
            }
            n[i] = (int)r;
        }
        if (!live) continue;
        u16* out = (val ? a.V : a.K) + ((long)t * a.G + g) * D + 2 * lane;
        *reinterpret_cast<u32u*>(out) = (uint32_t)y[0] | (uint32_t)y[1] << 16;
        *reinterpret_cast<u32u*>(out + D2) = (uint32_t)y[2] | (uint32_t)y[3] << 16;
        if (!keep) continue;
        const long head = page * a.G + g;
        const uint8_t b0 = (uint8_t)(n[0] | n[1] << 4), b1 = (uint8_t)(n[2] | n[3] << 4);
        // (token off: K's row of D2 bytes; V's byte off % 16 of every 16 in its block)
        uint8_t* c = (val ? a.Vc : a.Kc) + (head * a.P + (val ? off & ~15 : off)) * D2 + (val ? off & 15 : 0);
        c[lane * (val ? 16 : 1)] = b0;
        c[(D2 / 2 + lane) * (val ? 16 : 1)] = b1;
        if (lane == 0) {
            u16* s = (val ? a.Vs : a.Ks) + (head * a.P + off) * 2;
            s[0] = bad ? (u16)0x7e00 : f2h(lo);
            s[1] = bad ? (u16)0x7e00 : f2h((float)(range / 15.0));
        }
    }
}

// Workgroups of rows: at most 2^20 of them, which go on to later rows.
unsigned row_grid(long rows, int rpb) { return (unsigned)std::min((rows + rpb - 1) / rpb, 1L << 20); }

// The threads and register chunks of a row of K: f(NT, CH). CHUNKS: the most chunks a thread holds;
// quantize's rows stream faster with four loads a thread in flight (4096 x 5632 256 threads of 4 / 384 of 2 15.9 /
// 18.6 us), the norms', three times the registers, with two (512 x 8192 256 of 4 / 512 of 2 9.8 / 8.5).
template <int CHUNKS, class F>
void by_length(int K, F f) {
    auto go = [&](auto nt, auto ch) { f(nt, ch); };
#define Q_ROWS(NT, CH) go(std::integral_constant<int, NT>{}, std::integral_constant<int, CH>{})
    if (K <= 512) Q_ROWS(64, 1);
    else if (K <= 1024) Q_ROWS(64, 2);
    else if (K <= 2048) Q_ROWS(256, 1);
    else if (K <= 4096) Q_ROWS(256, 2);
    else if constexpr (CHUNKS == 4) {
        if (K <= 8192) Q_ROWS(256, 4);
        else if (K <= 16384) Q_ROWS(512, 4);
        else Q_ROWS(1024, 0);
    } else {
        if (K <= 6144) Q_ROWS(384, 2);
        else if (K <= 8192) Q_ROWS(512, 2);
        else if (K <= 12288) Q_ROWS(768, 2);
        else if (K <= 16384) Q_ROWS(1024, 2);
        else Q_ROWS(1024, 0);
    }
#undef Q_ROWS
}

int check_rows(const TslKernel& k, const char* rows, const char* cols) {
    if (k.dim(rows) > INT_MAX || k.dim(cols) > INT_MAX - 65536)
        return tsl_fail(-2, "quant/" + k.name + ": at most 2^31 - 1 rows of 2^31 - 65537 columns");
    return 0;
}

template <bool ADD>
int run_rmsnorm_q8(TslKernel& k, const u16* X, const uint64_t* a, hipStream_t s) {
    const int M = k.dim("T"), K = k.dim("Dm");
    if (M == 0) return 0;
    by_length<2>(K, [&](auto nt, auto ch) {
        constexpr int NT = decltype(nt)::value, CH = decltype(ch)::value, RPB = NT < 256 ? 256 / NT : 1;
        hipLaunchKernelGGL((rmsnorm_q8_kernel<NT, CH, ADD>), dim3(row_grid(M, RPB)), dim3(NT * RPB), 0, s, X,
                           P<float>(a[0]), P<u16>(a[1]), P<int8_t>(a[2]), P<float>(a[3]), M, K, arg_f32(a[4]));
    });
    return TSL_LAUNCHED("quant rmsnorm");
}

template <bool TABLE>
int run_kv_write(const KvArgs& r, int64_t D, hipStream_t s) {
    const int lanes = (int)std::min<long>(512, (2L * r.G * (D / 4) + 63) / 64 * 64);
    switch (D) {
        case 16: hipLaunchKernelGGL((kv_write_q4_kernel<16, TABLE>), dim3(r.T), dim3(lanes), 0, s, r); break;
        case 32: hipLaunchKernelGGL((kv_write_q4_kernel<32, TABLE>), dim3(r.T), dim3(lanes), 0, s, r); break;
        case 64: hipLaunchKernelGGL((kv_write_q4_kernel<64, TABLE>), dim3(r.T), dim3(lanes), 0, s, r); break;
        default: hipLaunchKernelGGL((kv_write_q4_kernel<128, TABLE>), dim3(r.T), dim3(lanes), 0, s, r); break;
    }
    return TSL_LAUNCHED("quant kv_write");
}

int table_bits(int T) {  // 2 T to 4 T places
    int bits = 1;
    while ((1L << bits) < 2L * T) bits++;
    return bits;
}

}  // namespace

int setup_quantize(TslKernel& k) { return check_rows(k, "M", "K"); }
int setup_rmsnorm_q8(TslKernel& k) {
    if (k.dim("Dm") == 0) return tsl_fail(-2, "quant/" + k.name + ": rows of 0 columns");
    return check_rows(k, "T", "Dm");
}

int launch_quantize(TslKernel& k, const uint64_t* a, hipStream_t s) {
    const int M = k.dim("M"), K = k.dim("K");
    if (M == 0) return 0;
    by_length<4>(K, [&](auto nt, auto ch) {
        constexpr int NT = decltype(nt)::value, CH = decltype(ch)::value, RPB = NT < 256 ? 256 / NT : 1;
        hipLaunchKernelGGL((quantize_kernel<NT, CH>), dim3(row_grid(M, RPB)), dim3(NT * RPB), 0, s, P<u16>(a[0]),
                           P<int8_t>(a[1]), P<float>(a[2]), M, K);
    });
    return TSL_LAUNCHED("quant quantize");
}

int launch_rmsnorm_q8(TslKernel& k, const uint64_t* a, hipStream_t s) { return run_rmsnorm_q8<false>(k, nullptr, a, s); }
int launch_add_rmsnorm_q8(TslKernel& k, const uint64_t* a, hipStream_t s) {
    return run_rmsnorm_q8<true>(k, P<u16>(a[0]), a + 1, s);
}

// The 4-bit cache's shape: D 16, 32, 64 or 128, D2 = D / 2 bytes a token, whole
// blocks of 16 tokens a page.
int check_cache_q4(const TslKernel& k) {
    const int64_t D = k.dim("D"), P = k.dim("P");
    if (D != 16 && D != 32 && D != 64 && D != 128)
        return tsl_fail(-2, "quant/" + k.name + ": head dimension " + std::to_string(D) + " unsupported (16, 32, 64 or 128)");
    if (k.dim("D2") * 2 != D) return tsl_fail(-2, "quant/" + k.name + ": D2 must be D / 2");
    if (P % 16 != 0) return tsl_fail(-2, "quant/" + k.name + ": pages must hold a multiple of 16 tokens");
    if (P > (1 << 30)) return tsl_fail(-2, "quant/" + k.name + ": pages hold at most 2^30 tokens");
    if (k.dim("PB") * 16 != P) return tsl_fail(-2, "quant/" + k.name + ": PB must be P / 16");
    if (k.dim("G") <= 0 || k.dim("NP") > INT_MAX || k.dim("G") > INT_MAX)
        return tsl_fail(-2, "quant/" + k.name + ": G and NP must be positive and below 2^31");
    return 0;
}

int setup_kv_write_q4(TslKernel& k) {
    if (int r = check_cache_q4(k)) return r;
    if (k.dim("W") < 2 * k.dim("G") * k.dim("D"))
        return tsl_fail(-2, "quant/kv_write: rows of W = " + std::to_string(k.dim("W")) + " hold no 2 G D keys and values");
    if (k.dim("T") >= (1 << 23) || k.dim("W") > INT_MAX || k.dim("NPOS") > INT_MAX)
        return tsl_fail(-2, "quant/kv_write: tokens below 2^23 and sizes below 2^31");
    return k.dim("T") > LOOK ? tsl_scratch(k, sizeof(unsigned long long) << table_bits((int)k.dim("T"))) : 0;
}

int launch_kv_write_q4(TslKernel& k, const uint64_t* a, hipStream_t s) {
    KvArgs r{};
    r.T = k.dim("T"), r.W = k.dim("W"), r.NPOS = k.dim("NPOS"), r.G = k.dim("G"), r.P = k.dim("P");
    r.NS = k.dim("NP") * k.dim("P");
    r.QKV = P<u16>(a[0]), r.pos = P<int>(a[1]), r.slot = P<int>(a[2]), r.Cs = P<float>(a[3]), r.Sn = P<float>(a[4]);
    r.Kc = P<uint8_t>(a[5]), r.Vc = P<uint8_t>(a[6]), r.Ks = P<u16>(a[7]), r.Vs = P<u16>(a[8]);
    r.K = P<u16>(a[9]), r.V = P<u16>(a[10]);
    if (r.T == 0) return 0;
    if (r.T > LOOK) {
        r.last = static_cast<unsigned long long*>(k.scratch), r.bits = table_bits(r.T);
        const unsigned clear = (unsigned)std::min<long>(1024, ((1L << (r.bits - 1)) + 255) / 256);
        hipLaunchKernelGGL(kv_clear_kernel, dim3(clear), dim3(256), 0, s, r);
        if (int e = TSL_LAUNCHED("quant kv_write table")) return e;
        hipLaunchKernelGGL(kv_last_kernel, dim3((unsigned)((r.T + 255) / 256)), dim3(256), 0, s, r);
        if (int e = TSL_LAUNCHED("quant kv_write table")) return e;
    }
    return r.last ? run_kv_write<true>(r, k.dim("D"), s) : run_kv_write<false>(r, k.dim("D"), s);
}
