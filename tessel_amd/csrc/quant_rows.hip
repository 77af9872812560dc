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

// The code of p in a row whose largest magnitude is top > 0: t = 127 p / top
// from inv = 127 / top, its whole number by adding 1.5 2^23 (f32) or rint
// (f64). NEAR bounds t's error (127 x 3 half-ulps, doubled); closer to a tie
// than that, 254 |p| is compared with (2 k + 1) top: p and top of 11 bits
// (f16) give 19-bit products, exact in f32; products of f32 and f16 (35
// bits) give 43-bit ones, exact in f64.
template <class F>
struct Code8;
template <>
struct Code8<float> {
    float top, inv;
    TSL_DEV explicit Code8(float t) : top(t), inv(t > 0.0f ? 127.0f / t : 0.0f) {}
    TSL_DEV int operator()(float p) const {
        constexpr float NEAR = 5e-5f;
        const float t = p * inv;
        float n = __builtin_rintf(t);
        if (__builtin_fabsf(t - n) > 0.5f - NEAR) {
            const float k = __builtin_floorf(__builtin_fabsf(t)), a = 254.0f * __builtin_fabsf(p), b = (2.0f * k + 1.0f) * top;
            const float m = a > b ? k + 1.0f : a < b ? k : 2.0f * __builtin_rintf(0.5f * (k + 0.5f));
            n = __builtin_copysignf(m, p);
        }
        return (int)n;
    }
};
template <>
struct Code8<double> {
    double top, inv;
    TSL_DEV explicit Code8(double t) : top(t), inv(t > 0.0 ? 127.0 / t : 0.0) {}
    TSL_DEV int operator()(double p) const {
        constexpr double NEAR = 1e-12;
        const double t = p * inv;
        double n = __builtin_rint(t);
        if (__builtin_fabs(t - n) > 0.5 - NEAR) {
            const double k = __builtin_floor(__builtin_fabs(t)), a = 254.0 * __builtin_fabs(p), b = (2.0 * k + 1.0) * top;
            const double m = a > b ? k + 1.0 : a < b ? k : 2.0 * __builtin_rint(0.5 * (k + 0.5));
            n = __builtin_copysign(m, p);
        }
        return (int)n;
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

// 8 codes as bytes, to row Q at column c of K (8-byte stores at any
// alignment; element by element where the chunk crosses the row's end).
TSL_DEV void store_codes(int8_t* q, int c, int K, const int (&n)[8]) {
    if (c + 8 <= K) {
        u32x2 v;
#pragma unroll
        for (int h = 0; h < 2; h++)
            v[h] = (uint32_t)(n[4 * h] & 255) | (uint32_t)(n[4 * h + 1] & 255) << 8 | (uint32_t)(n[4 * h + 2] & 255) << 16 |
                   (uint32_t)n[4 * h + 3] << 24;
        *reinterpret_cast<u32x2u*>(q + c) = v;
    } else {
#pragma unroll
        for (int e = 0; e < 8; e++)
            if (c + e < K) q[c + e] = (int8_t)n[e];
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
            int n[8];
#pragma unroll
            for (int e = 0; e < 8; e++) n[e] = bad ? 0 : code(h2f(half_of(w, e)));
            if (c < K) store_codes(Q + row * K, c, K, n);
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
            int n[8];
#pragma unroll
            for (int e = 0; e < 8; e++) n[e] = bad ? 0 : code((double)rr[e] * (double)h2f(half_of(ww, e)));
            if (c < K) store_codes(Q + row * K, c, K, n);
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

// kv_write: llm/kv_write's rotated keys and values, into K and V [T, G, D] as there
// and into the cache in 4 bits. A workgroup per (token, keys or values); D / 4
// lanes a head: lane j holds channels 2j, 2j + 1 and their rotary partners D/2
// on, which are the byte pairs j and D/4 + j.
struct KvArgs {
    const u16* QKV;
    const int *pos, *slot;
    const float *Cs, *Sn;
    uint8_t *Kc, *Vc;
    u16 *Ks, *Vs, *K, *V;
    int T, W, NPOS, G, P;
    long NS;
};

template <int D>
__global__ __launch_bounds__(256) void kv_write_q4_kernel(KvArgs a) {
    constexpr int D2 = D / 2, LPH = D / 4;
    const int t = blockIdx.x;
    const bool val = blockIdx.y;  // values (else keys)
    const int p = a.pos[t], at = a.slot[t];
    // Rows that name one slot: the last is kept. Every thread looks at its share of the later rows.
    bool later = false;
    for (int u = t + 1 + threadIdx.x; u < a.T; u += blockDim.x) later = later || a.slot[u] == at;
    const bool keep = !__syncthreads_or(later) && at >= 0 && at < a.NS;
    const int lane = threadIdx.x % LPH;
    const long page = keep ? at / a.P : 0;
    const int off = keep ? at % a.P : 0;
    // Every thread goes round as often (the reductions below take whole wavefronts).
    const int nh = blockDim.x / LPH;
    for (int g0 = 0; g0 < a.G; g0 += nh) {
        const int g = g0 + threadIdx.x / LPH;
        const bool live = g < a.G;
        const u16* x = a.QKV + (long)t * a.W + (a.W - (val ? 1L : 2L) * a.G * D) + (long)(live ? g : 0) * D;
        u16 y[4];
        if (val) {
#pragma unroll
            for (int i = 0; i < 2; i++) y[i] = x[2 * lane + i], y[2 + i] = x[D2 + 2 * lane + i];
        } else {
            const bool pin = p >= 0 && p < a.NPOS;
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const float c = pin ? a.Cs[(long)p * D2 + 2 * lane + i] : 0.0f;
                const float s = pin ? a.Sn[(long)p * D2 + 2 * lane + i] : 0.0f;
                rope_rotate(h2f(x[2 * lane + i]), h2f(x[D2 + 2 * lane + i]), c, s, y[i], y[2 + i]);
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
        auto both = [&](float l, float h) { lo = fminf(lo, l), hi = fmaxf(hi, h); };
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
                const double k = __builtin_floor(q), l = 30.0 * d, h = (2.0 * k + 1.0) * range;
                r = l > h ? k + 1.0 : l < h ? k : 2.0 * __builtin_rint(0.5 * (k + 0.5));
            }
            n[i] = (int)r;
        }
        if (!live) continue;
        u16* out = (val ? a.V : a.K) + ((long)t * a.G + g) * D;
#pragma unroll
        for (int i = 0; i < 2; i++) out[2 * lane + i] = y[i], out[D2 + 2 * lane + i] = y[2 + i];
        if (!keep) continue;
        const long head = page * a.G + g;
        const uint8_t b0 = (uint8_t)(n[0] | n[1] << 4), b1 = (uint8_t)(n[2] | n[3] << 4);
        if (val) {
            uint8_t* c = a.Vc + (head * (a.P / 16) + off / 16) * (D2 * 16) + off % 16;
            c[lane * 16] = b0;
            c[(D2 / 2 + lane) * 16] = b1;
        } else {
            uint8_t* c = a.Kc + (head * a.P + off) * D2;
            c[lane] = b0;
            c[D2 / 2 + lane] = b1;
        }
        if (lane == 0) {
            u16* s = (val ? a.Vs : a.Ks) + (head * a.P + off) * 2;
            s[0] = bad ? (u16)0x7e00 : f2h(lo);
            s[1] = bad ? (u16)0x7e00 : f2h((float)(range / 15.0));
        }
    }
}

// Workgroups of rows: at most 2^20 of them, which go on to later rows.
unsigned row_grid(long rows, int rpb) { return (unsigned)std::min((rows + rpb - 1) / rpb, 1L << 20); }

// The threads and register chunks of a row of K: f(NT, CH).
template <class F>
void by_length(int K, F f) {
    if (K <= 512) f(std::integral_constant<int, 64>{}, std::integral_constant<int, 1>{});
    else if (K <= 1024) f(std::integral_constant<int, 64>{}, std::integral_constant<int, 2>{});
    else if (K <= 2048) f(std::integral_constant<int, 256>{}, std::integral_constant<int, 1>{});
    else if (K <= 4096) f(std::integral_constant<int, 256>{}, std::integral_constant<int, 2>{});
    else if (K <= 8192) f(std::integral_constant<int, 256>{}, std::integral_constant<int, 4>{});
    else if (K <= 16384) f(std::integral_constant<int, 1024>{}, std::integral_constant<int, 2>{});
    else f(std::integral_constant<int, 1024>{}, std::integral_constant<int, 0>{});
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
    by_length(K, [&](auto nt, auto ch) {
        constexpr int NT = decltype(nt)::value, CH = decltype(ch)::value, RPB = NT < 256 ? 256 / NT : 1;
        hipLaunchKernelGGL((rmsnorm_q8_kernel<NT, CH, ADD>), dim3(row_grid(M, RPB)), dim3(NT * RPB), 0, s, X,
                           P<float>(a[0]), P<u16>(a[1]), P<int8_t>(a[2]), P<float>(a[3]), M, K, arg_f32(a[4]));
    });
    return TSL_LAUNCHED("quant rmsnorm");
}

}  // namespace

int check_quantize(TslKernel& k) { return check_rows(k, "M", "K"); }
int check_rmsnorm_q8(TslKernel& k) {
    if (k.dim("Dm") == 0) return tsl_fail(-2, "quant/" + k.name + ": rows of 0 columns");
    return check_rows(k, "T", "Dm");
}

int launch_quantize(TslKernel& k, const uint64_t* a, hipStream_t s) {
    const int M = k.dim("M"), K = k.dim("K");
    if (M == 0) return 0;
    by_length(K, [&](auto nt, auto ch) {
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
    if (k.dim("PB") * 16 != P) return tsl_fail(-2, "quant/" + k.name + ": PB must be P / 16");
    if (k.dim("G") <= 0 || k.dim("NP") > INT_MAX || k.dim("G") > INT_MAX)
        return tsl_fail(-2, "quant/" + k.name + ": G and NP must be positive and below 2^31");
    return 0;
}

int check_kv_write_q4(TslKernel& k) {
    if (int r = check_cache_q4(k)) return r;
    if (k.dim("W") < 2 * k.dim("G") * k.dim("D"))
        return tsl_fail(-2, "quant/kv_write: rows of W = " + std::to_string(k.dim("W")) + " hold no 2 G D keys and values");
    if (k.dim("T") > INT_MAX || k.dim("W") > INT_MAX || k.dim("NPOS") > INT_MAX)
        return tsl_fail(-2, "quant/kv_write: sizes must be below 2^31");
    return 0;
}

int launch_kv_write_q4(TslKernel& k, const uint64_t* a, hipStream_t s) {
    KvArgs r{};
    r.T = k.dim("T"), r.W = k.dim("W"), r.NPOS = k.dim("NPOS"), r.G = k.dim("G"), r.P = k.dim("P");
    r.NS = k.dim("NP") * k.dim("P");
    r.QKV = P<u16>(a[0]), r.pos = P<int>(a[1]), r.slot = P<int>(a[2]), r.Cs = P<float>(a[3]), r.Sn = P<float>(a[4]);
    r.Kc = P<uint8_t>(a[5]), r.Vc = P<uint8_t>(a[6]), r.Ks = P<u16>(a[7]), r.Vs = P<u16>(a[8]);
    r.K = P<u16>(a[9]), r.V = P<u16>(a[10]);
    if (r.T == 0) return 0;
    const int D = k.dim("D"), lanes = r.G * (D / 4) > 256 ? 256 : (r.G * (D / 4) + 63) / 64 * 64;
    switch (D) {
        case 16: hipLaunchKernelGGL(kv_write_q4_kernel<16>, dim3(r.T, 2), dim3(lanes), 0, s, r); break;
        case 32: hipLaunchKernelGGL(kv_write_q4_kernel<32>, dim3(r.T, 2), dim3(lanes), 0, s, r); break;
        case 64: hipLaunchKernelGGL(kv_write_q4_kernel<64>, dim3(r.T, 2), dim3(lanes), 0, s, r); break;
        default: hipLaunchKernelGGL(kv_write_q4_kernel<128>, dim3(r.T, 2), dim3(lanes), 0, s, r); break;
    }
    return TSL_LAUNCHED("quant kv_write");
}
