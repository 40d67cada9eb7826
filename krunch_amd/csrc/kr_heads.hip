// WKV with heads: a matrix state [D, D] per head of D = 64 or 128 channels, one
// decay and one bonus per head.
//
//   y_t = r_t (S + u k_t' v_t);   S <- e^w S + k_t' v_t        (w <= 0)
//
// Two forms. The recurrent one runs token by token in fp32 (k v is exact in
// fp32), so T tokens in one call have the bits of T calls. The chunked one takes
// 64 tokens at a time, with products on v_mfma_f32_16x16x32_f16: inside a chunk
//   y_i = e^(wi) r_i S + sum_{j<i} (r_i k_j) e^(w(i-j-1)) v_j + u (r_i k_i) v_i
//   S  <- e^(wn) S + sum_j k_j' (e^(w(n-1-j)) v_j)             (n tokens)
// r, k, v enter the matrix units as they are; the three fp32 quantities that do
// too, (r k) e^.., e^.. v and S, go in as two fp16 parts, high and low, scaled by
// a power of two to 2^14: 22 bits of each value, and 2^-38 of the largest
// one of a row (r k), a column (v) or 16 columns (S).
#include "kr_common.h"
#include "kr_wave.h"
#include "krunch_hip.h"

namespace {

constexpr float kLog2e = 0x1.715476p+0f;
constexpr int kChunk = 64;

struct HeadArgs {
    const kr_half* r;
    const kr_half* k;
    const kr_half* v;
    long long ldr, ldk, ldv;      // elements between tokens; a head's D are contiguous
    const float* decay;           // [H] w
    const float* first;           // [H] u
    const int32_t* lens;          // [B] tokens of each stream (null: T)
    float* state;                 // [B, H, D, D]
    kr_half* y;
    long long ldy;
    float* seg_state;             // [segments, B, H, D, D] (time split)
    int B, T, H;
    int seg_tokens, segments;     // segments of the time axis (1: none)
};

// log2 of the decay; w above 0 counts as 0 (and NaN stays).
__device__ __forceinline__ float decay_log2(float w) { return w > 0.0f ? 0.0f : w * kLog2e; }
// e^(w n), n >= 0; 1 at n = 0 whatever w is (-inf: no memory).
__device__ __forceinline__ float decay_pow(float w2, int n) {
    return n == 0 ? 1.0f : __builtin_amdgcn_exp2f(w2 * (float)n);
}
__device__ __forceinline__ int stream_tokens(const HeadArgs& g, int b) {
    if (!g.lens) return g.T;
    const int n = g.lens[b];
    return n < 0 ? 0 : n < g.T ? n : g.T;
}

// ---------------------------------------------------------------------------
// Recurrent form. A wave has 16 columns of a head's state in registers: lane
// l the columns 4 (l % 4) .. + 3 of rows D/16 (l / 4) .. + D/16 - 1, so y is
// summed over a lane's rows and then over 16 lanes, with no LDS.
// ---------------------------------------------------------------------------
template <int D>
__global__ void __launch_bounds__(4 * D) heads_step_kernel(HeadArgs g) {
    constexpr int R = D / 16;
    typedef kr_half rows_t __attribute__((ext_vector_type(R)));
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int h = blockIdx.x % g.H, b = blockIdx.x / g.H;
    const int m0 = 16 * wave + 4 * (lane & 3), n0 = R * (lane >> 2);
    const int T = stream_tokens(g, b);
    const float w2 = decay_log2(g.decay[h]), u = g.first[h];
    const float f = __builtin_amdgcn_exp2f(w2);
    float* st = g.state + ((size_t)blockIdx.x * D + n0) * D + m0;
    const size_t row0 = (size_t)b * g.T;
    const kr_half* rp = g.r + row0 * g.ldr + h * D + n0;
    const kr_half* kp = g.k + row0 * g.ldk + h * D + n0;
    const kr_half* vp = g.v + row0 * g.ldv + h * D + m0;
    kr_half* yp = g.y + row0 * g.ldy + h * D + m0;
    if (T > 0) {
        kr_float4 S[R];
        #pragma unroll
        for (int i = 0; i < R; i++) S[i] = *reinterpret_cast<const kr_float4*>(st + i * D);
        rows_t rn = *reinterpret_cast<const rows_t*>(rp), kn = *reinterpret_cast<const rows_t*>(kp);
        kr_half4 vn = *reinterpret_cast<const kr_half4*>(vp);
        for (int t = 0; t < T; t++) {
            const rows_t rt = rn, kt = kn;
            const kr_half4 vt = vn;
            if (t + 1 < T) {
                rp += g.ldr;
                kp += g.ldk;
                vp += g.ldv;
                rn = *reinterpret_cast<const rows_t*>(rp);
                kn = *reinterpret_cast<const rows_t*>(kp);
                vn = *reinterpret_cast<const kr_half4*>(vp);
            }
            kr_float4 y = kr_float4{0, 0, 0, 0};
            #pragma unroll
            for (int i = 0; i < R; i++) {
                #pragma unroll
                for (int c = 0; c < 4; c++) {
                    const float kv = (float)kt[i] * (float)vt[c];
                    y[c] = __builtin_fmaf((float)rt[i], __builtin_fmaf(u, kv, S[i][c]), y[c]);
                    S[i][c] = __builtin_fmaf(f, S[i][c], kv);
                }
            }
            #pragma unroll
            for (int c = 0; c < 4; c++) {
                y[c] += kr_xor<4>(y[c]);
                y[c] += kr_xor<8>(y[c]);
                y[c] += kr_xor<16>(y[c]);
                y[c] += kr_xor<32>(y[c]);
            }
            if (lane < 4)
                *reinterpret_cast<kr_half4*>(yp) =
                    kr_half4{kr_f16(y[0]), kr_f16(y[1]), kr_f16(y[2]), kr_f16(y[3])};
            yp += g.ldy;
        }
        #pragma unroll
        for (int i = 0; i < R; i++) *reinterpret_cast<kr_float4*>(st + i * D) = S[i];
    }
    if (lane < 4)
        for (int t = T; t < g.T; t++, yp += g.ldy)
            *reinterpret_cast<kr_half4*>(yp) = kr_half4{0, 0, 0, 0};
}

// ---------------------------------------------------------------------------
// Chunked form: a workgroup of 4 waves has one head of one stream (or one
// segment of its time axis) and walks its chunks.
// ---------------------------------------------------------------------------

// Powers of two that bring a largest value x to 2^13..2^14, and back. Zero and
// values under 2^-113 count as 2^-113; infinities and NaN pass through.
__device__ __forceinline__ void power_scale(float x, float& up, float& down) {
    int e = (int)(__float_as_uint(x) >> 23);
    e = e < 14 ? 14 : e;
    up = __uint_as_float((uint32_t)(267 - e) << 23);
    down = __uint_as_float((uint32_t)(e - 13) << 23);
}

// LDS tiles in 16-byte units. Token-major [64][D]: unit c of token t. Channel-
// major [D][64]: unit c (8 tokens) of channel n. The XORs keep the 8 lanes of a
// 16-byte access, and the writes of the transposed tiles, on different banks.
template <int D>
__device__ __forceinline__ int tok_unit(int t, int c) { return t * (D / 8) + (c ^ (t & (D / 8 - 1))); }
__device__ __forceinline__ int chan_unit(int n, int c) { return n * 8 + (c ^ ((n ^ (n >> 3)) & 7)); }

template <int D>
struct ChunkShared {
    kr_half8 r[kChunk * D / 8], k[kChunk * D / 8];     // token-major
    kr_half8 kt[D * 8], vt[D * 8];                     // channel-major
    kr_half8 ph[kChunk * 8], pl[kChunk * 8];           // [i][j], units of 8 j
    float pdown[kChunk];
};

// SUM: only the state that a segment's tokens add to zero.
template <int D, bool SUM>
__global__ void __launch_bounds__(256) heads_chunk_kernel(HeadArgs g) {
    constexpr int KS = D / 32;            // k-steps over the channels
    constexpr int MC = D / 64;            // 16-column tiles of a wave
    constexpr int NP = D / 64;            // token pairs a thread stages
    __shared__ ChunkShared<D> sh;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int l16 = lane & 15, q4 = lane >> 4;
    const int head = blockIdx.x, h = head % g.H, b = head / g.H, seg = blockIdx.y;
    const int heads = gridDim.x;
    const int t_begin = seg * g.seg_tokens;
    const int t_end = g.T - t_begin < g.seg_tokens ? g.T : t_begin + g.seg_tokens;
    const int live = stream_tokens(g, b);
    const int n_tok = live < t_begin ? 0 : (live < t_end ? live : t_end) - t_begin;
    const float w2 = decay_log2(g.decay[h]);
    const size_t row0 = (size_t)b * g.T + t_begin;

    // state: column m = D/4 wave + 16 c + l16; S[c][2s], S[c][2s + 1] hold rows
    // 32 s + 8 q4 + r and + 4, so that the pair is the operand of k-step s
    kr_float4 S[MC][2 * KS];
    const size_t state_at = (size_t)(8 * q4) * D + (D / 4) * wave + l16;
    const float* s_in = nullptr;
    if (!SUM)
        s_in = (g.segments > 1 ? g.seg_state + ((size_t)seg * heads + head) * D * D
                               : g.state + (size_t)head * D * D) + state_at;
    #pragma unroll
    for (int c = 0; c < MC; c++)
        #pragma unroll
        for (int s = 0; s < KS; s++)
            #pragma unroll
            for (int e = 0; e < 8; e++)
                S[c][2 * s + e / 4][e % 4] = SUM ? 0.0f : s_in[(size_t)(32 * s + e) * D + 16 * c];

    // what a thread stages: tokens 2p, 2p + 1 (p = p0 + 16 i ...), 8 channels
    const int ng = tid % (D / 8), p0 = tid / (D / 8);
    constexpr int PSTEP = 256 / (D / 8);
    kr_half8 rr[NP][2], kk[NP][2], vv[NP][2];
    auto fetch = [&](int t0) {
        #pragma unroll
        for (int i = 0; i < NP; i++)
            #pragma unroll
            for (int e = 0; e < 2; e++) {
                const int t = t0 + 2 * (p0 + PSTEP * i) + e;
                const kr_half8 zero = {0, 0, 0, 0, 0, 0, 0, 0};
                if (!SUM) rr[i][e] = zero;
                kk[i][e] = vv[i][e] = zero;
                if (t < n_tok) {
                    const size_t row = row0 + t;
                    const int o = h * D + 8 * ng;
                    if (!SUM) rr[i][e] = *reinterpret_cast<const kr_half8*>(g.r + row * g.ldr + o);
                    kk[i][e] = *reinterpret_cast<const kr_half8*>(g.k + row * g.ldk + o);
                    vv[i][e] = *reinterpret_cast<const kr_half8*>(g.v + row * g.ldv + o);
                }
            }
    };

    // decay factors of this lane. P tile (i-tile = wave, rows j): i = 16 wave +
    // l16, j = 16 jt + 4 q4 + r; e^(w(i-j-1)) = e^(w(i-16(jt+1))) e^(w(15-4 q4-r))
    // below the diagonal tile
    float p_far[3], p_near[4], p_diag[4], y_dec[4], v_dec[2 * 8];
    const float u = SUM ? 0.0f : g.first[h];
    if (!SUM) {
        #pragma unroll
        for (int jt = 0; jt < 3; jt++)
            p_far[jt] = jt < wave ? decay_pow(w2, 16 * (wave - jt - 1) + l16) : 0.0f;
        #pragma unroll
        for (int r = 0; r < 4; r++) {
            const int d = l16 - (4 * q4 + r);
            p_near[r] = decay_pow(w2, 15 - (4 * q4 + r));
            p_diag[r] = d > 0 ? decay_pow(w2, d - 1) : d == 0 ? u : 0.0f;
            y_dec[r] = decay_pow(w2, 16 * r + l16);
        }
        if ((wave & 1) == 0) {            // the half k-step right of the diagonal tile
            const int i = 16 * wave + l16, j = 16 * (wave + 1) + 4 * q4;
            kr_half4* ph = reinterpret_cast<kr_half4*>(sh.ph + chan_unit(i, j / 8)) + (j / 4 & 1);
            kr_half4* pl = reinterpret_cast<kr_half4*>(sh.pl + chan_unit(i, j / 8)) + (j / 4 & 1);
            *ph = *pl = kr_half4{0, 0, 0, 0};
        }
    }
    auto set_v_dec = [&](int n) {         // e^(w(n-1-j)), j = 32 s + 8 q4 + e
        #pragma unroll
        for (int i = 0; i < 16; i++) {
            const int left = n - 1 - (32 * (i / 8) + 8 * q4 + i % 8);
            v_dec[i] = left >= 0 ? decay_pow(w2, left) : 0.0f;
        }
    };
    set_v_dec(kChunk);

    fetch(0);
    for (int t0 = 0; t0 < n_tok; t0 += kChunk) {
        const int n = n_tok - t0 < kChunk ? n_tok - t0 : kChunk;
        if (n < kChunk) set_v_dec(n);
        #pragma unroll
        for (int i = 0; i < NP; i++) {
            const int p = p0 + PSTEP * i;
            #pragma unroll
            for (int e = 0; e < 2; e++) {
                if (!SUM) {
                    sh.r[tok_unit<D>(2 * p + e, ng)] = rr[i][e];
                    sh.k[tok_unit<D>(2 * p + e, ng)] = kk[i][e];
                }
            }
            typedef kr_half half2v __attribute__((ext_vector_type(2)));
            #pragma unroll
            for (int e = 0; e < 8; e++) {
                const int c = chan_unit(8 * ng + e, p / 4) * 4 + p % 4;
                reinterpret_cast<half2v*>(sh.kt)[c] = half2v{kk[i][0][e], kk[i][1][e]};
                reinterpret_cast<half2v*>(sh.vt)[c] = half2v{vv[i][0][e], vv[i][1][e]};
            }
        }
        if (t0 + kChunk < n_tok) fetch(t0 + kChunk);
        __syncthreads();
        if (!SUM) {
            // P' tiles of i-tile `wave`: rows j, columns i
            kr_half8 ri[KS];
            #pragma unroll
            for (int s = 0; s < KS; s++) ri[s] = sh.r[tok_unit<D>(16 * wave + l16, 4 * s + q4)];
            kr_float4 P[4];
            float big = 0.0f;
            #pragma unroll
            for (int jt = 0; jt < 4; jt++) {
                if (jt > wave) break;
                P[jt] = kr_float4{0, 0, 0, 0};
                #pragma unroll
                for (int s = 0; s < KS; s++)
                    P[jt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                        sh.k[tok_unit<D>(16 * jt + l16, 4 * s + q4)], ri[s], P[jt], 0, 0, 0);
                #pragma unroll
                for (int r = 0; r < 4; r++) {
                    P[jt][r] *= jt == wave ? p_diag[r] : p_far[jt < 3 ? jt : 0] * p_near[r];
                    big = fmaxf(big, fabsf(P[jt][r]));
                }
            }
            big = fmaxf(big, kr_xor<16>(big));
            big = fmaxf(big, kr_xor<32>(big));
            float up, down;
            power_scale(big, up, down);
            const int i = 16 * wave + l16;
            if (q4 == 0) sh.pdown[i] = down;
            #pragma unroll
            for (int jt = 0; jt < 4; jt++) {
                if (jt > wave) break;
                kr_half4 hi, lo;
                #pragma unroll
                for (int r = 0; r < 4; r++) {
                    const float x = P[jt][r] * up;
                    hi[r] = kr_f16(x);
                    lo[r] = kr_f16(x - (float)hi[r]);
                }
                const int at = chan_unit(i, 2 * jt + q4 / 2);
                reinterpret_cast<kr_half4*>(sh.ph + at)[q4 & 1] = hi;
                reinterpret_cast<kr_half4*>(sh.pl + at)[q4 & 1] = lo;
            }
            __syncthreads();
        }
        #pragma unroll
        for (int c = 0; c < MC; c++) {
            const int m = (D / 4) * wave + 16 * c + l16;
            kr_half8 vc[2];
            #pragma unroll
            for (int s = 0; s < 2; s++) vc[s] = sh.vt[chan_unit(m, 4 * s + q4)];
            if (!SUM) {
                float big = 0.0f;
                #pragma unroll
                for (int s = 0; s < 2 * KS; s++)
                    #pragma unroll
                    for (int r = 0; r < 4; r++) big = fmaxf(big, fabsf(S[c][s][r]));
                big = kr_wave_reduce(big, [](float x, float y) { return fmaxf(x, y); });
                float up, down;
                power_scale(big, up, down);
                kr_half8 sh_hi[KS], sh_lo[KS];
                #pragma unroll
                for (int s = 0; s < KS; s++)
                    #pragma unroll
                    for (int e = 0; e < 8; e++) {
                        const float x = S[c][2 * s + e / 4][e % 4] * up;
                        sh_hi[s][e] = kr_f16(x);
                        sh_lo[s][e] = kr_f16(x - (float)sh_hi[s][e]);
                    }
                // y': rows m, columns i
                #pragma unroll
                for (int it = 0; it < 4; it++) {
                    kr_float4 from_s = {0, 0, 0, 0}, inside = {0, 0, 0, 0};
                    #pragma unroll
                    for (int s = 0; s < KS; s++) {
                        const kr_half8 x = sh.r[tok_unit<D>(16 * it + l16, 4 * s + q4)];
                        from_s = __builtin_amdgcn_mfma_f32_16x16x32_f16(sh_hi[s], x, from_s, 0, 0, 0);
                        from_s = __builtin_amdgcn_mfma_f32_16x16x32_f16(sh_lo[s], x, from_s, 0, 0, 0);
                    }
                    #pragma unroll
                    for (int s = 0; s < 1 + it / 2; s++) {
                        const int at = chan_unit(16 * it + l16, 4 * s + q4);
                        inside = __builtin_amdgcn_mfma_f32_16x16x32_f16(vc[s], sh.ph[at], inside, 0, 0, 0);
                        inside = __builtin_amdgcn_mfma_f32_16x16x32_f16(vc[s], sh.pl[at], inside, 0, 0, 0);
                    }
                    const int i = 16 * it + l16;
                    const float fs = down * y_dec[it], fp = sh.pdown[i];
                    kr_half4 y;
                    #pragma unroll
                    for (int r = 0; r < 4; r++)
                        y[r] = kr_f16(__builtin_fmaf(inside[r], fp, from_s[r] * fs));
                    if (i < n)
                        *reinterpret_cast<kr_half4*>(g.y + (row0 + t0 + i) * g.ldy + h * D +
                                                     (D / 4) * wave + 16 * c + 4 * q4) = y;
                }
            }
            // S <- e^(wn) S + k' (e^.. v): v in two parts, scaled by its column
            float x[16], big = 0.0f;
            #pragma unroll
            for (int i = 0; i < 16; i++) {
                x[i] = (float)vc[i / 8][i % 8] * v_dec[i];
                big = fmaxf(big, fabsf(x[i]));
            }
            big = fmaxf(big, kr_xor<16>(big));
            big = fmaxf(big, kr_xor<32>(big));
            float up, down;
            power_scale(big, up, down);
            kr_half8 hi[2], lo[2];
            #pragma unroll
            for (int i = 0; i < 16; i++) {
                const float z = x[i] * up;
                hi[i / 8][i % 8] = kr_f16(z);
                lo[i / 8][i % 8] = kr_f16(z - (float)hi[i / 8][i % 8]);
            }
            const float keep = decay_pow(w2, n);
            #pragma unroll
            for (int st = 0; st < 2 * KS; st++) {
                // row l16 of the tile is channel 32 (st / 2) + 8 (l16 / 4) + 4 (st % 2) + l16 % 4
                const int ch = 32 * (st / 2) + 8 * (l16 >> 2) + 4 * (st % 2) + (l16 & 3);
                kr_float4 add = {0, 0, 0, 0};
                #pragma unroll
                for (int s = 0; s < 2; s++) {
                    const kr_half8 kc = sh.kt[chan_unit(ch, 4 * s + q4)];
                    add = __builtin_amdgcn_mfma_f32_16x16x32_f16(kc, hi[s], add, 0, 0, 0);
                    add = __builtin_amdgcn_mfma_f32_16x16x32_f16(kc, lo[s], add, 0, 0, 0);
                }
                #pragma unroll
                for (int r = 0; r < 4; r++)
                    S[c][st][r] = __builtin_fmaf(add[r], down, keep * S[c][st][r]);
            }
        }
        __syncthreads();
    }

    // the segment's sum goes to the next one's slot; the last segment has the state
    float* s_out = nullptr;
    if (SUM) s_out = g.seg_state + ((size_t)(seg + 1) * heads + head) * D * D;
    else if (seg == g.segments - 1) s_out = g.state + (size_t)head * D * D;
    if (s_out) {
        s_out += state_at;
        #pragma unroll
        for (int c = 0; c < MC; c++)
            #pragma unroll
            for (int s = 0; s < KS; s++)
                #pragma unroll
                for (int e = 0; e < 8; e++)
                    s_out[(size_t)(32 * s + e) * D + 16 * c] = S[c][2 * s + e / 4][e % 4];
    }
    if (!SUM)
        for (int i = n_tok * (D / 8) + tid; i < (t_end - t_begin) * (D / 8); i += 256)
            *reinterpret_cast<kr_half8*>(g.y + (row0 + i / (D / 8)) * g.ldy + h * D + 8 * (i % (D / 8))) =
                kr_half8{0, 0, 0, 0, 0, 0, 0, 0};
}

// Slot s of seg_state, which holds what segment s - 1 adds, becomes the state
// at the start of segment s.
template <int D>
__global__ void __launch_bounds__(256) heads_join_kernel(HeadArgs g) {
    const int heads = g.B * g.H;
    const size_t at = (size_t)blockIdx.x * 256 + threadIdx.x;      // float4 of all heads
    const int head = (int)(at / (D * D / 4));
    const int live = stream_tokens(g, head / g.H);
    const float w2 = decay_log2(g.decay[head % g.H]);
    const size_t slot = (size_t)heads * (D * D / 4);
    kr_float4* seg = reinterpret_cast<kr_float4*>(g.seg_state) + at;
    kr_float4 s = reinterpret_cast<const kr_float4*>(g.state)[at];
    seg[0] = s;
    for (int i = 1; i < g.segments; i++) {
        const int before = (i - 1) * g.seg_tokens;
        const int n = live < before ? 0 : live - before < g.seg_tokens ? live - before : g.seg_tokens;
        const float keep = decay_pow(w2, n);
        const kr_float4 add = seg[i * slot];
        #pragma unroll
        for (int r = 0; r < 4; r++) s[r] = __builtin_fmaf(keep, s[r], add[r]);
        seg[i * slot] = s;
    }
}

// Tokens up to which the chunked form is the recurrent one, too.
constexpr int kStepTokens = 16;
// Workgroups that a time split aims for, and the fewest tokens of a segment.
constexpr int kSplitGroups = 512, kSplitTokens = 128;

void split_time(long long heads, int T, int& tokens, int& segments) {
    long long n = (kSplitGroups + heads - 1) / heads;
    const long long most = (T + kSplitTokens - 1) / kSplitTokens;
    if (n > most) n = most;
    tokens = (int)(((T + n - 1) / n + kChunk - 1) / kChunk * kChunk);
    segments = (T + tokens - 1) / tokens;
}

template <int D>
int launch(HeadArgs& g, bool chunked, hipStream_t s) {
    const int heads = g.B * g.H;
    if (!chunked || g.T <= kStepTokens) {
        heads_step_kernel<D><<<heads, 4 * D, 0, s>>>(g);
    } else if (g.segments == 1) {
        heads_chunk_kernel<D, false><<<heads, 256, 0, s>>>(g);
    } else {
        heads_chunk_kernel<D, true><<<dim3(heads, g.segments - 1), 256, 0, s>>>(g);
        KR_LAUNCHED();
        heads_join_kernel<D><<<heads * (D * D / 1024), 256, 0, s>>>(g);
        KR_LAUNCHED();
        heads_chunk_kernel<D, false><<<dim3(heads, g.segments), 256, 0, s>>>(g);
    }
    KR_LAUNCHED();
    return KR_OK;
}

bool shape_ok(int B, int T, int H, int D) {
    return B >= 0 && T >= 0 && H >= 1 && (D == 64 || D == 128) &&
           (long long)B * H * (D * D / 1024) <= 0x7fffffff && T <= 1 << 30;
}

}  // namespace

extern "C" {

size_t kr_wkv_heads_workspace_bytes(int B, int T, int H, int D) {
    if (!shape_ok(B, T, H, D) || B == 0 || T <= kStepTokens) return 0;
    int tokens, segments;
    split_time((long long)B * H, T, tokens, segments);
    return segments == 1 ? 0 : (size_t)segments * B * H * D * D * sizeof(float);
}

int kr_wkv_heads(int B, int T, int H, int D, const uint16_t* r, long long ldr, const uint16_t* k,
                 long long ldk, const uint16_t* v, long long ldv, const float* decay,
                 const float* first, const int32_t* lens, float* state, uint16_t* y, long long ldy,
                 int chunked, void* ws, size_t ws_bytes, void* stream) {
    KR_REQUIRE(shape_ok(B, T, H, D), "kr_wkv_heads: bad shape B=%d T=%d H=%d D=%d (D: 64 or 128)", B, T,
               H, D);
    const long long C = (long long)H * D;
    KR_REQUIRE(ldr >= C && ldk >= C && ldv >= C && ldy >= C && (ldr | ldk | ldv | ldy) % 8 == 0,
               "kr_wkv_heads: token strides must be multiples of 8 and at least H * D = %lld", C);
    if (B == 0 || T == 0) return KR_OK;
    KR_REQUIRE(r && k && v && decay && first && state && y, "kr_wkv_heads: null pointer");
    KR_REQUIRE((((uintptr_t)r | (uintptr_t)k | (uintptr_t)v | (uintptr_t)state | (uintptr_t)y) & 15) == 0,
               "kr_wkv_heads: r, k, v, state and y must be 16-byte aligned");
    HeadArgs g{};
    g.r = reinterpret_cast<const kr_half*>(r);
    g.k = reinterpret_cast<const kr_half*>(k);
    g.v = reinterpret_cast<const kr_half*>(v);
    g.ldr = ldr;
    g.ldk = ldk;
    g.ldv = ldv;
    g.decay = decay;
    g.first = first;
    g.lens = lens;
    g.state = state;
    g.y = reinterpret_cast<kr_half*>(y);
    g.ldy = ldy;
    g.B = B;
    g.T = T;
    g.H = H;
    g.segments = 1;
    g.seg_tokens = T;
    if (chunked && T > kStepTokens) {
        split_time((long long)B * H, T, g.seg_tokens, g.segments);
        const size_t need = kr_wkv_heads_workspace_bytes(B, T, H, D);
        KR_REQUIRE(need == 0 || (ws && ws_bytes >= need && ((uintptr_t)ws & 15) == 0),
                   "kr_wkv_heads: workspace of %zu bytes, %zu needed (16-byte aligned)", ws_bytes, need);
        g.seg_state = reinterpret_cast<float*>(ws);
    }
    return D == 64 ? launch<64>(g, chunked != 0, kr_stream(stream))
                   : launch<128>(g, chunked != 0, kr_stream(stream));
}

}  // extern "C"
