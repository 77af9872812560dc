// Decode attention over the paged cache in 4 bits (quant/decode_attention; not a
// .tl kernel): llm/decode_attention with K and V given as 4-bit codes and a
// pair (lowest value, step) for each token and kv head, value = low + step code.
//   Kc [NP, G, P, D/2]:       byte j of a token: channels 2j (low nibble), 2j + 1
//   Vc [NP, G, P/16, D/2, 16]: the same bytes, 16 tokens of a channel pair together
//   Ks, Vs [NP, G, P, 2]:     (low, step), f16
// With low and step factored out, a score is
//   q . k = step (q . n) + low sum(q)
// and an output sum(p v) = sum((p step) n) + sum(p low), so only the small whole
// numbers n go through the products. A page outside [0, NP) reads as zeros and an
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
    int CT;       // tokens per chunk
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
    const int c = blockIdx.x % a.NCH;
    const long bg = blockIdx.x / a.NCH;
    const int g = bg % a.G, b = bg / a.G;
    const int n = tokens_of(a, b);
    const int nact = max(1, (int)(((long)n + a.CT - 1) / a.CT));  // (at most NCH)
    if (c >= nact) return;
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
            vlow = h2f(a.Vs[2 * at]);
            vstep = h2f(a.Vs[2 * at + 1]);
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
                const float n0 = v & 15, n1 = v >> 4;
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

// Joins a (sequence, query head)'s chunks in order; a wavefront each.
template <int D>
__global__ __launch_bounds__(64) void decode_q4_join(Q4Args a, int qpg) {
    const int h = blockIdx.x % a.H, g = h / qpg, i = h % qpg;
    const long b = blockIdx.x / a.H;
    const int nact = max(1, (int)(((long)tokens_of(a, b) + a.CT - 1) / a.CT));
    const float* p = a.part + ((b * a.G + g) * a.NCH * qpg + i) * (2L + D);
    const long next = (long)qpg * (2 + D);
    float m = -INFINITY;
    for (int c = 0; c < nact; c++) m = fmaxf(m, p[c * next]);
    for (int d = threadIdx.x; d < D; d += 64) {
        float l = 0.0f, v = 0.0f;
        for (int c = 0; c < nact; c++) {
            const float f = __builtin_amdgcn_exp2f(p[c * next] - m);
            l += p[c * next + 1] * f;
            v += p[c * next + 2 + d] * f;
        }
        a.O[(b * a.H + h) * D + d] = f2h(v / l);
    }
}

// Tokens a chunk: 256 at least, and about 2048 workgroups at the table's full length.
int chunk_tokens(const TslKernel& k) {
    const int64_t bg = std::max<int64_t>(1, k.dim("B") * k.dim("G")), most = k.dim("MP") * k.dim("P");
    return (int)std::min<int64_t>(std::max<int64_t>(256, (most * bg / 2048 + 255) / 256 * 256), 1 << 24);
}
int nchunks(const TslKernel& k) {
    const int64_t most = k.dim("MP") * k.dim("P"), ct = chunk_tokens(k);
    return (int)std::max<int64_t>(1, (most + ct - 1) / ct);
}

template <int D>
int run_q4(const Q4Args& a, int qpg, hipStream_t s) {
    const unsigned grid = (unsigned)((long)a.B * a.G * a.NCH);
    switch (qpg) {
        case 1: hipLaunchKernelGGL((decode_q4_any<D, 1>), dim3(grid), dim3(256), 0, s, a); break;
        case 2: hipLaunchKernelGGL((decode_q4_any<D, 2>), dim3(grid), dim3(256), 0, s, a); break;
        case 4: hipLaunchKernelGGL((decode_q4_any<D, 4>), dim3(grid), dim3(256), 0, s, a); break;
        case 8: hipLaunchKernelGGL((decode_q4_any<D, 8>), dim3(grid), dim3(256), 0, s, a); break;
        default: hipLaunchKernelGGL((decode_q4_any<D, 16>), dim3(grid), dim3(256), 0, s, a); break;
    }
    int r = TSL_LAUNCHED("quant decode_attention");
    if (r || a.NCH == 1) return r;
    hipLaunchKernelGGL(decode_q4_join<D>, dim3((unsigned)((long)a.B * a.H)), dim3(64), 0, s, a, qpg);
    return TSL_LAUNCHED("quant decode_attention join");
}

}  // namespace

int check_decode_q4(TslKernel& k) {
    if (int r = check_cache_q4(k)) return r;
    const int64_t H = k.dim("H"), G = k.dim("G"), B = k.dim("B"), MP = k.dim("MP");
    if (H % G != 0) return tsl_fail(-2, "quant/decode_attention: H must be a multiple of G");
    const int64_t qpg = H / G;
    if (qpg != 1 && qpg != 2 && qpg != 4 && qpg != 8 && qpg != 16)
        return tsl_fail(-2, "quant/decode_attention: H / G must be 1, 2, 4, 8 or 16");
    if (MP > INT_MAX / k.dim("P") || B * H > (1 << 24) || B * G * nchunks(k) > (1 << 24))
        return tsl_fail(-2, "quant/decode_attention: at most 2^31 - 1 tokens a table and 2^24 (sequence, head, chunk)s");
    return 0;
}

int prepare_decode_q4(TslKernel& k) {
    if (nchunks(k) > 1) {
        const size_t bytes = (size_t)k.dim("B") * k.dim("H") * nchunks(k) * (2 + k.dim("D")) * sizeof(float);
        if (bytes && tsl_hip_check(hipMalloc(&k.scratch, bytes), "quant/decode_attention scratch")) return -1;
        k.scratch_bytes = bytes;
    }
    return 0;
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
    a.NCH = nchunks(k), a.CT = chunk_tokens(k);
    a.part = reinterpret_cast<float*>(k.scratch);
    if (a.B == 0) return 0;
    const int qpg = a.H / a.G;
    switch (k.dim("D")) {
        case 16: return run_q4<16>(a, qpg, s);
        case 32: return run_q4<32>(a, qpg, s);
        case 64: return run_q4<64>(a, qpg, s);
        default: return run_q4<128>(a, qpg, s);
    }
}
