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
// one of a row (r k) or of a column (v, S).
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
// Bound, for one token: the state, read and written once. Measured on MI355X, heads
// of 64: 512 streams x 12 heads 38 us (203 MB, 5.4 TB/s; a copy runs at 5.1), one
// stream 3.0. For many: at few streams a token's chain (1 x 256 tokens 118 us, 64 x 256
// 251: 0.5 and 1.0 us a token), at many the VALU (512 x 64 tokens 400 us, 6.2 a token; the
// bytes would take 78).
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
// Chunked form: a workgroup has one head of one stream (or one segment of its time
// axis) and walks its chunks, a wave for each 16 columns of the state, which stays
// in the wave's registers as the matrix unit leaves it: as such it is the operand
// of r S, too. r, k and v of a chunk are read ahead into registers, then go to
// LDS by token (r, k) and transposed by channel (k, v). The first four waves make
// (r k') e^.. for 16 tokens each, halves of it above the diagonal left out.
// Bound: with many heads, the VALU work of taking values apart (about 500
// instructions a chunk and wave beside 50 products) and the three barriers, with 3
// workgroups a CU for D = 64 and one for 128; with few heads, latency. Measured on
// MI355X, heads of 64: 256 x 1024 tokens x 12 heads 393 us (1.71 GB, 4.4 TB/s), 128
// streams of 256..1024 155 us (640 MB, 4.1 TB/s; 10 more in the order they come), 1 x
// 4096 24; heads of 128: 128 x 1024 x 6 278 us (3.2 TB/s), 1 x 1777 x 8 28.
// ---------------------------------------------------------------------------

// Powers of two that bring a largest value x to 2^13..2^14, and back. Zero and
// values under 2^-113 count as 2^-113; infinities and NaN pass through.
__device__ __forceinline__ void power_scale(float x, float& up, float& down) {
    int e = (int)(__float_as_uint(x) >> 23);
    e = e < 14 ? 14 : e;
    up = __uint_as_float((uint32_t)(267 - e) << 23);
    down = __uint_as_float((uint32_t)(e - 13) << 23);
}

// x as a high and a low fp16 part.
__device__ __forceinline__ void two_parts(float x, kr_half& hi, kr_half& lo) {
    __asm__("" : "+v"(x));       // or x is made twice, in 7 spilled registers (400 -> 473 us)
    hi = (kr_half)x;
    lo = (kr_half)(x - (float)hi);
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
__global__ void __launch_bounds__(4 * D, D == 64 ? 3 : 2) heads_chunk_kernel(HeadArgs g) {
    constexpr int KS = D / 32;            // k-steps over the channels
    __shared__ ChunkShared<D> sh;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int l16 = lane & 15, q4 = lane >> 4;
    const int heads = gridDim.x, seg = blockIdx.y, h = blockIdx.x % g.H;
    int b = blockIdx.x / g.H;
    if (!SUM && g.lens && g.segments == 1 && g.B <= 4 * D) {
        // longest streams first, so that no long one is left for the end: thread i
        // ranks stream i (the sh.ph are written after the next barrier only)
        int* lens = reinterpret_cast<int*>(sh.ph);
        if (tid < g.B) lens[tid] = stream_tokens(g, tid);
        __syncthreads();
        int rank = 0;
        if (tid < g.B) {
            const int mine = lens[tid];
            #pragma unroll 8
            for (int j = 0; j < g.B; j++) rank += lens[j] > mine || (lens[j] == mine && j < tid);
            if (rank == b) reinterpret_cast<int*>(sh.pl)[0] = tid;
        }
        __syncthreads();
        b = __builtin_amdgcn_readfirstlane(reinterpret_cast<int*>(sh.pl)[0]);
        __syncthreads();
    }
    const int head = b * g.H + h;
    const int t_begin = seg * g.seg_tokens;
    const int t_end = g.T - t_begin < g.seg_tokens ? g.T : t_begin + g.seg_tokens;
    const int live = stream_tokens(g, b);
    const int n_tok = live < t_begin ? 0 : (live < t_end ? live : t_end) - t_begin;
    const float w2 = decay_log2(g.decay[h]);
    const size_t row0 = (size_t)b * g.T + t_begin;

    // state: column m = 16 wave + l16; S[2s], S[2s + 1] hold rows 32 s + 8 q4 + r and
    // + 4, so that the pair is the operand of k-step s
    kr_float4 S[2 * KS];
    const int m = 16 * wave + l16;
    const size_t state_at = (size_t)(8 * q4) * D + m;
    const float* s_in = nullptr;
    if (!SUM)
        s_in = (g.segments > 1 ? g.seg_state + ((size_t)seg * heads + head) * D * D
                               : g.state + (size_t)head * D * D) + state_at;
    #pragma unroll
    for (int s = 0; s < KS; s++)
        #pragma unroll
        for (int e = 0; e < 8; e++)
            S[2 * s + e / 4][e % 4] = SUM ? 0.0f : s_in[(size_t)(32 * s + e) * D];

    // what a thread stages: 8 channels of tokens 2p, 2p + 1
    const int ng = tid % (D / 8), p = tid / (D / 8);
    kr_half8 rr[2], kk[2], vv[2];
    const size_t first = row0 + 2 * p;
    const kr_half* rp = g.r + first * g.ldr + h * D + 8 * ng;
    const kr_half* kp = g.k + first * g.ldk + h * D + 8 * ng;
    const kr_half* vp = g.v + first * g.ldv + h * D + 8 * ng;
    auto fetch = [&](int t0) {            // in order of t0
        #pragma unroll
        for (int e = 0; e < 2; e++) {
            const kr_half8 zero = {0, 0, 0, 0, 0, 0, 0, 0};
            if (!SUM) rr[e] = zero;
            kk[e] = vv[e] = zero;
            if (t0 + 2 * p + e < n_tok) {
                if (!SUM) rr[e] = *reinterpret_cast<const kr_half8*>(rp + e * g.ldr);
                kk[e] = *reinterpret_cast<const kr_half8*>(kp + e * g.ldk);
                vv[e] = *reinterpret_cast<const kr_half8*>(vp + e * g.ldv);
            }
        }
        rp += kChunk * g.ldr;
        kp += kChunk * g.ldk;
        vp += kChunk * g.ldv;
    };
    kr_half* yp = g.y + (row0 + l16) * g.ldy + h * D + 16 * wave + 4 * q4;

    // decay factors of this lane. P tile (i-tile = wave, rows j): i = 16 wave +
    // l16, j = 16 jt + 4 q4 + r; e^(w(i-j-1)) = e^(w(i-16(jt+1))) e^(w(15-4 q4-r))
    // below the diagonal tile
    float p_far[3], p_near[4], p_diag[4], y_dec[4], v_dec[2 * 8];
    const float u = SUM ? 0.0f : g.first[h];
    if (!SUM) {
        #pragma unroll
        for (int jt = 0; jt < 3; jt++)
            p_far[jt] = jt < wave && wave < 4 ? decay_pow(w2, 16 * (wave - jt - 1) + l16) : 0.0f;
        #pragma unroll
        for (int r = 0; r < 4; r++) {
            const int d = l16 - (4 * q4 + r);
            p_near[r] = decay_pow(w2, 15 - (4 * q4 + r));
            p_diag[r] = d > 0 ? decay_pow(w2, d - 1) : d == 0 ? u : 0.0f;
            y_dec[r] = decay_pow(w2, 16 * r + l16);
        }
        if (wave == 0 || wave == 2) {     // the half k-step right of the diagonal tile
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
        // LDS addresses are made anew for each chunk: kept over the loop, they and
        // the reads moved up to them spill
        int l16 = lane & 15, q4 = lane >> 4;
        __asm__ volatile("" : "+v"(l16), "+v"(q4));
        if (n < kChunk) set_v_dec(n);
        typedef kr_half half2v __attribute__((ext_vector_type(2)));
        #pragma unroll
        for (int e = 0; e < 2; e++) {
            if (!SUM) {
                sh.r[tok_unit<D>(2 * p + e, ng)] = rr[e];
                sh.k[tok_unit<D>(2 * p + e, ng)] = kk[e];
            }
        }
        #pragma unroll
        for (int e = 0; e < 8; e++) {
            const int c = chan_unit(8 * ng + e, p / 4) * 4 + p % 4;
            reinterpret_cast<half2v*>(sh.kt)[c] = half2v{kk[0][e], kk[1][e]};
            reinterpret_cast<half2v*>(sh.vt)[c] = half2v{vv[0][e], vv[1][e]};
        }
        if (t0 + kChunk < n_tok) fetch(t0 + kChunk);
        __syncthreads();
        if (!SUM) {
            if (wave < 4) {
                // P' tiles of i-tile `wave`: rows j, columns i
                kr_half8 ri[KS];
                #pragma unroll
                for (int s = 0; s < KS; s++) ri[s] = sh.r[tok_unit<D>(16 * wave + l16, 4 * s + q4)];
                kr_float4 P[4];
                float big = 0.0f;
                #pragma unroll
                for (int jt = 0; jt < 4; jt++) {
                    P[jt] = kr_float4{0, 0, 0, 0};
                    if (jt > wave) continue;
                    #pragma unroll
                    for (int s = 0; s < KS; s++)
                        P[jt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                            sh.k[tok_unit<D>(16 * jt + l16, 4 * s + q4)], ri[s], P[jt], 0, 0, 0);
                    #pragma unroll
                    for (int r = 0; r < 4; r++) {
                        P[jt][r] *= jt == wave ? p_diag[r] : p_far[jt < 3 ? jt : 0] * p_near[r];
                        big = fmaxf(big, fabsf(P[jt][r]));
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
                big = fmaxf(big, kr_xor<16>(big));
                big = fmaxf(big, kr_xor<32>(big));
                float up, down;
                power_scale(big, up, down);
                const int i = 16 * wave + l16;
                if (q4 == 0) sh.pdown[i] = down;
                #pragma unroll
                for (int jt = 0; jt < 4; jt++) {
                    if (jt > wave) continue;
                    kr_half4 hi, lo;
                    #pragma unroll
                    for (int r = 0; r < 4; r++) {
                        kr_half a, b;
                        two_parts(P[jt][r] * up, a, b);
                        hi[r] = a;
                        lo[r] = b;
                    }
                    const int at = chan_unit(i, 2 * jt + q4 / 2);
                    reinterpret_cast<kr_half4*>(sh.ph + at)[q4 & 1] = hi;
                    reinterpret_cast<kr_half4*>(sh.pl + at)[q4 & 1] = lo;
                }
            }
            __syncthreads();
        }
        __builtin_amdgcn_sched_barrier(0);
        kr_half8 vc[2];
        #pragma unroll
        for (int s = 0; s < 2; s++) vc[s] = sh.vt[chan_unit(m, 4 * s + q4)];
        if (!SUM) {
            // a scale for each column, so that an infinite or a huge one changes no other
            float big = 0.0f;
            #pragma unroll
            for (int s = 0; s < 2 * KS; s++)
                #pragma unroll
                for (int r = 0; r < 4; r++) big = fmaxf(big, fabsf(S[s][r]));
            big = fmaxf(big, kr_xor<16>(big));
            big = fmaxf(big, kr_xor<32>(big));
            float up, down;
            power_scale(big, up, down);
            kr_half8 s_hi[KS], s_lo[KS];
            #pragma unroll
            for (int s = 0; s < KS; s++)
                #pragma unroll
                for (int e = 0; e < 8; e++) {
                    kr_half a, b;
                    two_parts(S[2 * s + e / 4][e % 4] * up, a, b);
                    s_hi[s][e] = a;
                    s_lo[s][e] = b;
                }
            kr_float4 down_m;              // of the rows m that this lane has of y'
            #pragma unroll
            for (int r = 0; r < 4; r++) down_m[r] = __shfl(down, 4 * q4 + r);
            __builtin_amdgcn_sched_barrier(0);
            // y': rows m, columns i
            #pragma unroll
            for (int it = 0; it < 4; it++) {
                kr_float4 from_s = {0, 0, 0, 0}, inside = {0, 0, 0, 0};
                #pragma unroll
                for (int s = 0; s < KS; s++) {
                    const kr_half8 x = sh.r[tok_unit<D>(16 * it + l16, 4 * s + q4)];
                    from_s = __builtin_amdgcn_mfma_f32_16x16x32_f16(s_hi[s], x, from_s, 0, 0, 0);
                    from_s = __builtin_amdgcn_mfma_f32_16x16x32_f16(s_lo[s], x, from_s, 0, 0, 0);
                }
                #pragma unroll
                for (int s = 0; s < 1 + it / 2; s++) {
                    const int at = chan_unit(16 * it + l16, 4 * s + q4);
                    inside = __builtin_amdgcn_mfma_f32_16x16x32_f16(vc[s], sh.ph[at], inside, 0, 0, 0);
                    inside = __builtin_amdgcn_mfma_f32_16x16x32_f16(vc[s], sh.pl[at], inside, 0, 0, 0);
                }
                const int i = 16 * it + l16;
                const float fp = sh.pdown[i];
                kr_half4 y;
                #pragma unroll
                for (int r = 0; r < 4; r++)
                    y[r] = kr_f16(__builtin_fmaf(inside[r], fp, from_s[r] * (down_m[r] * y_dec[it])));
                if (i < n)
                    *reinterpret_cast<kr_half4*>(yp + 16 * it * g.ldy) = y;
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        __builtin_amdgcn_sched_barrier(0);
        yp += kChunk * g.ldy;
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
            kr_half a, b;
            two_parts(x[i] * up, a, b);
            hi[i / 8][i % 8] = a;
            lo[i / 8][i % 8] = b;
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
            for (int r = 0; r < 4; r++) S[st][r] = __builtin_fmaf(add[r], down, keep * S[st][r]);
            if (st % 2) __builtin_amdgcn_sched_barrier(0);
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
        for (int s = 0; s < KS; s++)
            #pragma unroll
            for (int e = 0; e < 8; e++) s_out[(size_t)(32 * s + e) * D] = S[2 * s + e / 4][e % 4];
    }
    if (!SUM)
        for (int i = n_tok * (D / 8) + tid; i < (t_end - t_begin) * (D / 8); i += 4 * D)
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
    constexpr int kAhead = 8;             // or every step waits for memory (16: the same time)
    for (int i0 = 1; i0 < g.segments; i0 += kAhead) {
        kr_float4 add[kAhead];
        #pragma unroll
        for (int j = 0; j < kAhead; j++)
            if (i0 + j < g.segments) add[j] = seg[(i0 + j) * slot];
        #pragma unroll
        for (int j = 0; j < kAhead; j++) {
            const int i = i0 + j;
            if (i >= g.segments) break;
            const int before = (i - 1) * g.seg_tokens;
            const int n = live < before ? 0 : live - before < g.seg_tokens ? live - before : g.seg_tokens;
            const float keep = decay_pow(w2, n);
            #pragma unroll
            for (int r = 0; r < 4; r++) s[r] = __builtin_fmaf(keep, s[r], add[j][r]);
            seg[i * slot] = s;
        }
    }
}

// Tokens up to which the chunked form is the recurrent one, too. us, recurrent /
// chunked, 12 heads of 64: 8 tokens of 1 stream 6.1 / 6.7, of 64 13.4 / 13.2, of 512
// 64 / 62; 16 tokens 9.5 / 6.8, 20.7 / 13.2, 112 / 64.
constexpr int kStepTokens = 8;
// Workgroups that a time split aims for, and the fewest tokens of a segment. A split
// reads k and v twice and costs two launches. us, aiming for 256 / 512 / 1024: 32 x 512
// x 12 heads of 64 37.7 / 45.7 / 51.8, 16 x 1024 53 / 52 / 55, 16 x 1024 x 6 of 128 78 /
// 86 / 92; segments of 64 / 128 / 256 tokens: 1 x 256 x 12 12.6 / 15.9 / 15.3, 1 x 1777 x
// 8 of 128 28.6 / 31.7 / 42.2, 1 x 4096 x 12 26.5 / 26.5 / 29.2.
constexpr int kSplitGroups = 256, kSplitTokens = 64;

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
        heads_chunk_kernel<D, false><<<heads, 4 * D, 0, s>>>(g);
    } else {
        heads_chunk_kernel<D, true><<<dim3(heads, g.segments - 1), 4 * D, 0, s>>>(g);
        KR_LAUNCHED();
        heads_join_kernel<D><<<heads * (D * D / 1024), 256, 0, s>>>(g);
        KR_LAUNCHED();
        heads_chunk_kernel<D, false><<<dim3(heads, g.segments), 4 * D, 0, s>>>(g);
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
