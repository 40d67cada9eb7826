// The gated delta rule: a matrix state [D, D] per head of D = 64 or 128 channels, a
// decay and a write strength per token and head.
//
//   S <- e^g S;  u = beta (v - k S);  S <- S + k' u;  y = q S          (g <= 0)
//
// Two forms. The recurrent one runs token by token in fp32. The chunked one takes
// 64 tokens at a time: with a_i the sum of g to token i of the chunk and
//   A_ij = e^(a_i - a_j) k_i k_j' (j < i),  P_ij = e^(a_i - a_j) q_i k_j' (j <= i)
// what the tokens find different from the state, r = v - e^a k S - A u with u = beta r,
// is the solution of a triangular system, and
//   y = e^a q S + P u;   S <- e^a_end S + sum_j k_j' (e^(a_end - a_j) u_j).
// For a block of tokens r = X - N (beta X) with N = A (1 + beta A)^-1, strictly
// lower triangular: no division by beta, exact where beta is 0. N of 16 x 16
// blocks comes from forward substitution (powers of beta A would cancel where keys repeat), of
// 32 x 32 from two products; the two halves of a chunk are solved in turn.
//
// q, k, v enter the matrix units (v_mfma_f32_16x16x32_f16) as they are; fp32 values
// that do too, S, P, N, A and columns of beta X and u, go in as two fp16 parts, high
// and low, scaled by a power of two to 2^14: 22 bits of each value, and 2^-38 of
// the largest one of a row (P, N, A) or of a column (S, beta X, u).
#include "kr_common.h"
#include "kr_wave.h"
#include "krunch_hip.h"

namespace {

constexpr int kChunk = 64;

struct DeltaArgs {
    const kr_half* q;
    const kr_half* k;
    const kr_half* v;
    long long ldq, ldk, ldv;      // elements between tokens; a head's D are contiguous
    const float* gate;            // log decays, [B, T] by ldg, heads contiguous
    const float* beta;
    long long ldg, ldb;
    const int32_t* lens;          // [B] tokens of each stream (null: T)
    float* state;                 // [B, H, D, D]
    kr_half* y;                   // [B, T, H, D] by ldy
    long long ldy;
    float* before;                // STATES: [chunks + 1][heads][D][D], the state before each chunk
    float* diff;                  // STATES: [chunks][heads][64][D], r
    float* sums;                  // SUMS: [segments][heads][D][D] what a segment adds
    float* maps;                  // SUMS: [segments][heads][D][D] what it makes of a state
    float* starts;                // [segments][heads][D][D] (time split: the states at the starts)
    int B, T, H;
    int seg_chunks, segments;     // segments of the time axis (1: none)
};
enum { FORWARD, STATES, SUMS };   // what a walk over chunks leaves: y; states and r; sums or maps

__device__ __forceinline__ int stream_tokens(const int32_t* lens, int b, int T) {
    if (!lens) return T;
    const int n = lens[b];
    return n < 0 ? 0 : n < T ? n : T;
}

// log2 of a decay, sums of 64 of which stay finite: g above 0 counts as 0, below
// -10000 as that (both e^g are 0), NaN stays.
__device__ __forceinline__ double gate_log2(float g) {
    g = g > 0.0f ? 0.0f : g < -10000.0f ? -10000.0f : g;
    return (double)g * 0x1.71547652b82fep+0;
}

// ---------------------------------------------------------------------------
// Recurrent form. A wave has 16 columns of a head's state in registers: lane l the
// columns 4 (l % 4) .. + 3 of rows D/16 (l / 4) .. + D/16 - 1. k S, q S and k q' are
// summed together over a lane's rows and then over 16 lanes: y = q S + (q k') u.
// Bound, for one token: the state, read and written once. Measured on MI355X, heads of
// 64: 512 streams x 12 heads 32 us (203 MB, 6.3 TB/s), one stream 3.2 (a call 11, the
// host's). For many: a token's chain, 0.7 us.
// ---------------------------------------------------------------------------
template <int D>
__global__ void __launch_bounds__(4 * D) delta_step_kernel(DeltaArgs g) {
    constexpr int R = D / 16;
    typedef kr_half rows_t __attribute__((ext_vector_type(R)));
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int h = blockIdx.x % g.H, b = blockIdx.x / g.H;
    const int m0 = 16 * wave + 4 * (lane & 3), n0 = R * (lane >> 2);
    const int T = stream_tokens(g.lens, b, g.T);
    float* st = g.state + ((size_t)blockIdx.x * D + n0) * D + m0;
    const size_t row0 = (size_t)b * g.T;
    const kr_half* qp = g.q + row0 * g.ldq + h * D + n0;
    const kr_half* kp = g.k + row0 * g.ldk + h * D + n0;
    const kr_half* vp = g.v + row0 * g.ldv + h * D + m0;
    const float* gp = g.gate + row0 * g.ldg + h;
    const float* bp = g.beta + row0 * g.ldb + h;
    kr_half* yp = g.y + row0 * g.ldy + h * D + m0;
    if (T > 0) {
        kr_float4 S[R];
        #pragma unroll
        for (int i = 0; i < R; i++) S[i] = *reinterpret_cast<const kr_float4*>(st + i * D);
        rows_t qn = *reinterpret_cast<const rows_t*>(qp), kn = *reinterpret_cast<const rows_t*>(kp);
        kr_half4 vn = *reinterpret_cast<const kr_half4*>(vp);
        float gn = *gp, bn = *bp;
        for (int t = 0; t < T; t++) {
            const rows_t qt = qn, kt = kn;
            const kr_half4 vt = vn;
            const float f = __builtin_amdgcn_exp2f((float)gate_log2(gn)), beta = bn;
            if (t + 1 < T) {
                qp += g.ldq;
                kp += g.ldk;
                vp += g.ldv;
                gp += g.ldg;
                bp += g.ldb;
                qn = *reinterpret_cast<const rows_t*>(qp);
                kn = *reinterpret_cast<const rows_t*>(kp);
                vn = *reinterpret_cast<const kr_half4*>(vp);
                gn = *gp;
                bn = *bp;
            }
            kr_float4 kS = {0, 0, 0, 0}, qS = {0, 0, 0, 0};
            float kq = 0.0f;
            #pragma unroll
            for (int i = 0; i < R; i++) {
                kq = __builtin_fmaf((float)kt[i], (float)qt[i], kq);
                #pragma unroll
                for (int c = 0; c < 4; c++) {
                    S[i][c] *= f;
                    kS[c] = __builtin_fmaf((float)kt[i], S[i][c], kS[c]);
                    qS[c] = __builtin_fmaf((float)qt[i], S[i][c], qS[c]);
                }
            }
            kq += kr_xor<4>(kq);
            kq += kr_xor<8>(kq);
            kq += kr_xor<16>(kq);
            kq += kr_xor<32>(kq);
            kr_half4 y;
            #pragma unroll
            for (int c = 0; c < 4; c++) {
                kS[c] += kr_xor<4>(kS[c]);
                qS[c] += kr_xor<4>(qS[c]);
                kS[c] += kr_xor<8>(kS[c]);
                qS[c] += kr_xor<8>(qS[c]);
                kS[c] += kr_xor<16>(kS[c]);
                qS[c] += kr_xor<16>(qS[c]);
                kS[c] += kr_xor<32>(kS[c]);
                qS[c] += kr_xor<32>(qS[c]);
                const float u = beta * ((float)vt[c] - kS[c]);
                #pragma unroll
                for (int i = 0; i < R; i++) S[i][c] = __builtin_fmaf((float)kt[i], u, S[i][c]);
                y[c] = kr_f16(__builtin_fmaf(kq, u, qS[c]));
            }
            if (lane < 4) *reinterpret_cast<kr_half4*>(yp) = y;
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
// Parts of the chunked kernels.
// ---------------------------------------------------------------------------

// The lane, made anew: LDS addresses that follow from it are not kept over a chunk,
// where they and the reads moved up to them spill.
__device__ __forceinline__ int fresh(int lane) {
    __asm__ volatile("" : "+v"(lane));
    return lane;
}
// Nothing is moved over this, for the same reason.
__device__ __forceinline__ void phase() { __builtin_amdgcn_sched_barrier(0); }

// Powers of two that bring a largest value x to 2^13..2^14, and back. Zero and
// values under 2^-113 count as 2^-113; infinities and NaN pass through.
__device__ __forceinline__ void power_scale(float x, float& up, float& down) {
    int e = (int)(__float_as_uint(x) >> 23);
    e = e < 14 ? 14 : e;
    up = __uint_as_float((uint32_t)(267 - e) << 23);
    down = __uint_as_float((uint32_t)(e - 13) << 23);
}

// x up as a high and a low fp16 part (up a power of two: two instructions, since both
// are an fma rounded to fp16).
__device__ __forceinline__ void two_parts(float x, float up, kr_half& hi, kr_half& lo) {
    hi = (kr_half)__builtin_fmaf(x, up, 0.0f);
    lo = (kr_half)__builtin_fmaf(x, up, -(float)hi);
}

__device__ __forceinline__ float max_of_quarters(float x) {       // over lanes l % 16
    x = fmaxf(x, kr_xor<16>(x));
    return fmaxf(x, kr_xor<32>(x));
}

// 8 values of a column or row that 4 lanes (l / 16) hold, in two parts.
struct Parts8 {
    kr_half8 hi, lo;
};
__device__ __forceinline__ float largest8(const float (&x)[8], float big = 0.0f) {
    #pragma unroll
    for (int e = 0; e < 8; e++) big = fmaxf(big, fabsf(x[e]));
    return big;
}
__device__ __forceinline__ Parts8 parts8(const float (&x)[8], float up) {
    Parts8 p;
    #pragma unroll
    for (int e = 0; e < 8; e++) {
        kr_half a, b;
        two_parts(x[e], up, a, b);
        p.hi[e] = a;
        p.lo[e] = b;
    }
    return p;
}
__device__ __forceinline__ Parts8 scaled8(const float (&x)[8], float& down) {
    float up;
    power_scale(max_of_quarters(largest8(x)), up, down);
    return parts8(x, up);
}

__device__ __forceinline__ kr_float4 mfma(kr_half8 a, kr_half8 b, kr_float4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
// a (two parts) times b (two parts), without low x low.
__device__ __forceinline__ kr_float4 mfma3(kr_half8 ah, kr_half8 al, const Parts8& b, kr_float4 c) {
    c = mfma(al, b.hi, c);
    c = mfma(ah, b.lo, c);
    return mfma(ah, b.hi, c);
}

// LDS tiles in 16-byte units. Of tokens [64][D]: unit c of token t. Of pairs
// [64][64]: unit c (8 columns) of row i. The XORs keep the 8 lanes of a 16-byte access
// on different banks.
template <int D>
__device__ __forceinline__ int tok_unit(int t, int c) { return t * (D / 8) + (c ^ (t & (D / 8 - 1))); }
__device__ __forceinline__ int pair_unit(int i, int c) { return i * 8 + (c ^ ((i ^ (i >> 3)) & 7)); }

// Transposing reads of a token tile: 8 tokens (32 s + 8 (l / 16) ..) of 16 channels,
// one a lane. channels16: channel 16 tile + l % 16. channels_state: the channel of
// row l % 16 of state tile st, 32 (st / 2) + 8 (l % 16 / 4) + 4 (st % 2) + l % 4.
typedef short short4v __attribute__((__vector_size__(8)));
typedef __attribute__((address_space(3))) short4v lds_short4;
template <int D>
__device__ __forceinline__ kr_half8 read_tokens(const kr_half8* tile, int s, int unit, int half, int lane) {
    typedef kr_half half4v __attribute__((ext_vector_type(4)));
    const int t = 32 * s + 8 * (lane >> 4) + ((lane & 15) >> 2);
    const unsigned base = (unsigned)(uintptr_t)(__attribute__((address_space(3))) const char*)tile + 8 * half;
    const unsigned at0 = base + 16 * tok_unit<D>(t, unit), at1 = base + 16 * tok_unit<D>(t + 4, unit);
    const half4v a = __builtin_bit_cast(half4v, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4*)(uintptr_t)at0));
    const half4v b = __builtin_bit_cast(half4v, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4*)(uintptr_t)at1));
    return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
}
template <int D>
__device__ __forceinline__ kr_half8 channels16(const kr_half8* tile, int s, int t16, int lane) {
    return read_tokens<D>(tile, s, 2 * t16 + ((lane & 3) >> 1), lane & 1, lane);
}
template <int D>
__device__ __forceinline__ kr_half8 channels_state(const kr_half8* tile, int s, int st, int lane) {
    return read_tokens<D>(tile, s, 4 * (st >> 1) + (lane & 3), st & 1, lane);
}

// Per chunk: sums of log2 decays, and what follows from them. A decay between tokens of
// two tiles of 16 is one to the later tile's start times one from there, both at most
// 1: a product instead of an exponential a pair.
struct alignas(16) Gates {
    double a[kChunk];
    float e0[kChunk], e1[kChunk], beta[kChunk];   // e^a, e^(a_end - a), write strengths
    float from[kChunk];                           // from the start of the token's tile to it
    float to[3][kChunk];                          // from the token to the start of tile 1, 2, 3
    float all;                                    // e^a_end
};
// By one wave, lane = token.
__device__ __forceinline__ void make_gates(Gates& o, float gate, float beta, int lane) {
    double a = gate_log2(gate);
    #pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const double b = __shfl_up(a, d);
        if (lane >= d) a += b;
    }
    const double end = __shfl(a, 63), starts[3] = {__shfl(a, 15), __shfl(a, 31), __shfl(a, 47)};
    const double start = lane < 16 ? 0.0 : lane < 32 ? starts[0] : lane < 48 ? starts[1] : starts[2];
    o.a[lane] = a;
    o.e0[lane] = __builtin_amdgcn_exp2f((float)a);
    o.e1[lane] = __builtin_amdgcn_exp2f((float)(end - a));
    o.beta[lane] = beta;
    o.from[lane] = __builtin_amdgcn_exp2f((float)(a - start));
    #pragma unroll
    for (int i = 0; i < 3; i++) o.to[i][lane] = __builtin_amdgcn_exp2f((float)(starts[i] - a));
    if (lane == 63) o.all = __builtin_amdgcn_exp2f((float)end);
}
// e^(a_row - a_col) for 4 columns from `col`, of an earlier tile than row's, w.
__device__ __forceinline__ kr_float4 decays_to(const Gates& g, int w, float from_row, int col) {
    return *reinterpret_cast<const kr_float4*>(g.to[w - 1] + col) * from_row;
}
// The same for columns of a later tile ct, e^(a_col - a_row).
__device__ __forceinline__ kr_float4 decays_from(const Gates& g, int ct, int row, int col) {
    return *reinterpret_cast<const kr_float4*>(g.from + col) * g.to[ct - 1][row];
}

// The triangular matrices of a chunk as operands: rows i, units of 8 j. M holds N
// of the chunk's two halves in its diagonal 32 x 32 blocks and A below them. With
// TRANSPOSED, rows are j and units i, of all three.
constexpr int kWork = 36;             // floats of a row
struct Pairs {
    kr_half8 ph[kChunk * 8], pl[kChunk * 8];
    kr_half8 mh[kChunk * 8], ml[kChunk * 8];
    float p_down[kChunk], n_down[kChunk], a_down[kChunk];
    float work[2][32 * kWork];    // fp32 A, then N, of the two halves
};

__device__ __forceinline__ void store_parts4(kr_half8* hi, kr_half8* lo, int row, int col, kr_float4 x, float up) {
    kr_half4 h, l;
    #pragma unroll
    for (int r = 0; r < 4; r++) {
        kr_half a, b;
        two_parts(x[r], up, a, b);
        h[r] = a;
        l[r] = b;
    }
    const int at = pair_unit(row, col / 8);
    reinterpret_cast<kr_half4*>(hi + at)[col / 4 & 1] = h;
    reinterpret_cast<kr_half4*>(lo + at)[col / 4 & 1] = l;
}

// P (or P') of 16 rows by one wave, w = 0..3.
template <int D, bool TRANSPOSED>
__device__ __forceinline__ void make_p(Pairs& o, const kr_half8* q, const kr_half8* k, const Gates& gates, int w,
                                       int lane) {
    constexpr int KS = D / 32;
    phase();
    lane = fresh(lane);
    const int l16 = lane & 15, q4 = lane >> 4, row = 16 * w + l16;
    kr_half8 mine[KS];
    #pragma unroll
    for (int s = 0; s < KS; s++) mine[s] = (TRANSPOSED ? k : q)[tok_unit<D>(row, 4 * s + q4)];
    const double a = gates.a[row];
    const float from = gates.from[row];
    kr_float4 P[4];
    float big = 0.0f;
    // all four tiles, though those on one side of the diagonal are not used: their reads
    // and products are in flight together
    #pragma unroll
    for (int ct = 0; ct < 4; ct++) {
        P[ct] = kr_float4{0, 0, 0, 0};
        #pragma unroll
        for (int s = 0; s < KS; s++)
            P[ct] = mfma((TRANSPOSED ? q : k)[tok_unit<D>(16 * ct + l16, 4 * s + q4)], mine[s], P[ct]);
    }
    #pragma unroll
    for (int ct = 0; ct < 4; ct++) {
        const int col = 16 * ct + 4 * q4;
        if (ct == w) {
            #pragma unroll
            for (int r = 0; r < 4; r++) {
                const double d = TRANSPOSED ? gates.a[col + r] - a : a - gates.a[col + r];
                const bool on = TRANSPOSED ? col + r >= row : col + r <= row;
                P[ct][r] = on ? P[ct][r] * __builtin_amdgcn_exp2f((float)d) : 0.0f;
            }
        } else if (TRANSPOSED ? ct > w : ct < w) {
            P[ct] *= TRANSPOSED ? decays_from(gates, ct, row, col) : decays_to(gates, w, from, col);
        } else {
            P[ct] = kr_float4{0, 0, 0, 0};
        }
        #pragma unroll
        for (int r = 0; r < 4; r++) big = fmaxf(big, fabsf(P[ct][r]));
    }
    float up, down;
    power_scale(max_of_quarters(big), up, down);
    if (q4 == 0) o.p_down[row] = down;
    #pragma unroll
    for (int ct = 0; ct < 4; ct++) {
        // tiles of zeros inside a k-step of 32 are written, too
        if (TRANSPOSED ? ct / 2 < w / 2 : ct / 2 > w / 2) continue;
        store_parts4(o.ph, o.pl, row, 16 * ct + 4 * q4, P[ct], up);
    }
}

// 16 rows of k against 16 others: a tile of k k' with rows `col`.. and columns row..
template <int D>
__device__ __forceinline__ kr_float4 key_products(const kr_half8* k, int row0, int col0, int l16, int q4) {
    kr_float4 A = {0, 0, 0, 0};
    #pragma unroll
    for (int s = 0; s < D / 32; s++)
        A = mfma(k[tok_unit<D>(col0 + l16, 4 * s + q4)], k[tok_unit<D>(row0 + l16, 4 * s + q4)], A);
    return A;
}

// The diagonal tile w of A, fp32.
template <int D>
__device__ __forceinline__ void make_diagonal(Pairs& o, const kr_half8* k, const Gates& gates, int w, int lane) {
    phase();
    lane = fresh(lane);
    const int l16 = lane & 15, q4 = lane >> 4, row = 16 * w + l16, col = 16 * w + 4 * q4;
    kr_float4 A = key_products<D>(k, 16 * w, 16 * w, l16, q4);
    const double a = gates.a[row];
    #pragma unroll
    for (int r = 0; r < 4; r++) {
        const float e = __builtin_amdgcn_exp2f((float)(a - gates.a[col + r]));
        A[r] = col + r < row ? A[r] * e : 0.0f;
    }
    *reinterpret_cast<kr_float4*>(o.work[w / 2] + (row & 31) * kWork + (col & 31)) = A;
}

// The tile below it in a half, fp32.
template <int D>
__device__ __forceinline__ void make_half(Pairs& o, const kr_half8* k, const Gates& gates, int half, int lane) {
    phase();
    lane = fresh(lane);
    const int l16 = lane & 15, q4 = lane >> 4, w = 2 * half + 1, row = 16 * w + l16, col = 32 * half + 4 * q4;
    kr_float4 A = key_products<D>(k, 16 * w, 32 * half, l16, q4);
    A *= decays_to(gates, w, gates.from[row], col);
    *reinterpret_cast<kr_float4*>(o.work[half] + (16 + l16) * kWork + 4 * q4) = A;
}

// 16 rows of the block below the halves (w = 2, 3; transposed its columns, w = 0, 1), as operand.
template <int D, bool TRANSPOSED>
__device__ __forceinline__ void make_below(Pairs& o, const kr_half8* k, const Gates& gates, int w, int lane) {
    phase();
    lane = fresh(lane);
    const int l16 = lane & 15, q4 = lane >> 4, row = 16 * w + l16, c0 = TRANSPOSED ? 32 : 0;
    kr_float4 A[2];
    float big = 0.0f;
    #pragma unroll
    for (int ct = 0; ct < 2; ct++) A[ct] = key_products<D>(k, 16 * w, c0 + 16 * ct, l16, q4);
    #pragma unroll
    for (int ct = 0; ct < 2; ct++) {
        const int col = c0 + 16 * ct + 4 * q4;
        A[ct] *= TRANSPOSED ? decays_from(gates, 2 + ct, row, col) : decays_to(gates, w, gates.from[row], col);
        #pragma unroll
        for (int r = 0; r < 4; r++) big = fmaxf(big, fabsf(A[ct][r]));
    }
    float up, down;
    power_scale(max_of_quarters(big), up, down);
    if (q4 == 0) o.a_down[row] = down;
    #pragma unroll
    for (int ct = 0; ct < 2; ct++) store_parts4(o.mh, o.ml, row, c0 + 16 * ct + 4 * q4, A[ct], up);
}

__device__ __forceinline__ void wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// N of the four 16 x 16 diagonal blocks, in place of A, by one wave, 16 lanes each: row
// by row, N_t = A_t - sum_j A_tj (beta_j N_j); lane = column.
__device__ __forceinline__ void solve_16(Pairs& o, const Gates& gates, int lane) {
    phase();
    lane = fresh(lane);
    const int l16 = lane & 15, w = lane >> 4;
    float* block = o.work[w / 2] + 16 * (w & 1) * (kWork + 1);
    const float* beta = gates.beta + 16 * w;
    float N[16], bN[16];
    #pragma unroll
    for (int t = 0; t < 16; t++) {
        float x = block[kWork * t + l16];
        #pragma unroll
        for (int j4 = 0; j4 < t; j4 += 4) {
            const kr_float4 at = *reinterpret_cast<const kr_float4*>(block + kWork * t + j4);
            #pragma unroll
            for (int j = j4; j < j4 + 4 && j < t; j++) x = __builtin_fmaf(-at[j - j4], bN[j], x);
        }
        N[t] = x;
        bN[t] = beta[t] * x;
    }
    wave_sync();
    #pragma unroll
    for (int t = 0; t < 16; t++) block[kWork * t + l16] = N[t];
    wave_sync();
}

// The 16 x 16 block below in a half, by one wave: with Y = A10 - A10 (beta N00),
// N10 = Y - N11 (beta Y).
__device__ __forceinline__ void solve_32(Pairs& o, const Gates& gates, int half, int lane) {
    phase();
    lane = fresh(lane);
    const int l16 = lane & 15, q4 = lane >> 4;
    float* work = o.work[half];
    const float* beta = gates.beta + 32 * half;
    kr_float4 Y;
    #pragma unroll
    for (int r = 0; r < 4; r++) Y[r] = work[kWork * (16 + 4 * q4 + r) + l16];
    const kr_float4 a10 = *reinterpret_cast<const kr_float4*>(work + kWork * (16 + l16) + 4 * q4);
    const kr_float4 n11 = *reinterpret_cast<const kr_float4*>(work + kWork * (16 + l16) + 16 + 4 * q4);
    const kr_float4 b0 = *reinterpret_cast<const kr_float4*>(beta + 4 * q4);
    const kr_float4 b1 = *reinterpret_cast<const kr_float4*>(beta + 16 + 4 * q4);
    #pragma unroll
    for (int s = 0; s < 4; s++)
        Y = __builtin_amdgcn_mfma_f32_16x16x4f32(-a10[s], b0[s] * work[kWork * (4 * q4 + s) + l16], Y, 0, 0, 0);
    kr_float4 N = Y;
    #pragma unroll
    for (int s = 0; s < 4; s++) N = __builtin_amdgcn_mfma_f32_16x16x4f32(-n11[s], b1[s] * Y[s], N, 0, 0, 0);
    wave_sync();
    #pragma unroll
    for (int r = 0; r < 4; r++) work[kWork * (16 + 4 * q4 + r) + l16] = N[r];
    wave_sync();
}

// 16 rows of N of a half (columns for TRANSPOSED) as operands, by one wave.
template <bool TRANSPOSED>
__device__ __forceinline__ void store_n(Pairs& o, int w, int lane) {
    phase();
    lane = fresh(lane);
    const int l16 = lane & 15, q4 = lane >> 4, row = 16 * w + l16;
    const float* work = o.work[w / 2];
    float x[8];
    #pragma unroll
    for (int e = 0; e < 8; e++) {
        const int i = TRANSPOSED ? 8 * q4 + e : row & 31, j = TRANSPOSED ? row & 31 : 8 * q4 + e;
        x[e] = j < i ? work[kWork * i + j] : 0.0f;
    }
    float down;
    const Parts8 p = scaled8(x, down);
    if (q4 == 0) o.n_down[row] = down;
    const int at = pair_unit(row, 4 * (w / 2) + q4);
    o.mh[at] = p.hi;
    o.ml[at] = p.lo;
}

// All of them, by the workgroup's 4 or 8 waves; tokens and gates are in LDS, and the
// matrices are when it returns. One wave solves the diagonal tiles while the others make
// the rest. next(): for one wave meanwhile.
template <int D, bool TRANSPOSED, bool WITH_P, typename Next>
__device__ __forceinline__ void make_pairs(Pairs& o, const kr_half8* q, const kr_half8* k, const Gates& gates, int wave,
                                           int lane, Next next) {
    // rows of P by how many tiles they have, 1 to 4
    auto p_rows = [](int tiles) { return TRANSPOSED ? 4 - tiles : tiles - 1; };
    auto make_rows = [&](int w) { make_p<D, TRANSPOSED>(o, q, k, gates, w, lane); };
    if (wave < 4) make_diagonal<D>(o, k, gates, wave, lane);
    else if (WITH_P && wave >= 6) make_rows(p_rows(wave - 3));        // 4, 3
    __syncthreads();
    if (wave == 0) {
        solve_16(o, gates, lane);
    } else if (wave == 1) {
        make_half<D>(o, k, gates, 0, lane);
        if (D == 64 && WITH_P) make_rows(p_rows(4));
        else make_half<D>(o, k, gates, 1, lane);
    } else if (wave == 2) {
        make_below<D, TRANSPOSED>(o, k, gates, TRANSPOSED ? 0 : 2, lane);
        if (D == 64 && WITH_P) make_rows(p_rows(3));
        next();
    } else if (wave == 3) {
        make_below<D, TRANSPOSED>(o, k, gates, TRANSPOSED ? 1 : 3, lane);
        if (D == 64 && WITH_P) {
            make_half<D>(o, k, gates, 1, lane);
            make_rows(p_rows(2));
            make_rows(p_rows(1));
        }
    } else if (WITH_P && wave < 6) {
        make_rows(p_rows(wave - 3));                                  // 1, 2
    }
    __syncthreads();
    if (wave < 4) {
        // the rows that take the tile below wait for it
        if ((wave & 1) == (TRANSPOSED ? 0 : 1)) solve_32(o, gates, wave / 2, lane);
        store_n<TRANSPOSED>(o, wave, lane);
    }
    __syncthreads();
}

// Which stream this workgroup has: longest first, so that no long one is left for the end.
template <int THREADS>
__device__ __forceinline__ int ranked_stream(const int32_t* lens, int B, int T, int b, int* tmp) {
    const int tid = threadIdx.x;
    if (!lens || B > THREADS) return b;
    if (tid < B) tmp[tid] = stream_tokens(lens, tid, T);
    __syncthreads();
    int rank = 0;
    if (tid < B) {
        const int mine = tmp[tid];
        #pragma unroll 8
        for (int j = 0; j < B; j++) rank += tmp[j] > mine || (tmp[j] == mine && j < tid);
        if (rank == b) tmp[THREADS] = tid;
    }
    __syncthreads();
    b = __builtin_amdgcn_readfirstlane(tmp[THREADS]);
    __syncthreads();
    return b;
}

template <int D>
struct DeltaShared {
    kr_half8 q[kChunk * D / 8], k[kChunk * D / 8], v[kChunk * D / 8];      // by tokens
    Pairs pairs;
    Gates gates[2];
};

// ---------------------------------------------------------------------------
// Chunked form, forward: a workgroup has one head of one stream (or a segment of its
// time axis) and walks its chunks, a wave for each 16 columns of the state, which
// stays in the wave's registers as the matrix unit leaves it: as such it is the operand
// of k S and q S, and what they leave is the operand of the next product. A segment
// makes map S + sum of the state S at its start: SUMS gives one or the other, as the
// state that follows from the identity without values, or from zero.
// Bound: instructions issued, about 2,100 a chunk and wave (1,400 of them VALU, a third
// for taking values apart and scales), with 8 waves a CU: 72 KB of LDS a workgroup for D =
// 64, 96 for 128, allow no more; a wave alone issues one about every 8 cycles. Measured on
// MI355X, heads of 64: 128 streams of 256..1024 tokens x 12 heads 263-287 us (640 MB: 125 at
// a copy's rate; VALU 60% busy, matrix units 16%); a chunk alone 8 us, for D = 128 10.
// ---------------------------------------------------------------------------
template <int D, int MODE>
__device__ __forceinline__ void walk_chunks(const DeltaArgs& g, DeltaShared<D>& sh, int heads, int b, int h, int seg,
                                            bool map) {
    constexpr int KS = D / 32;            // k-steps over the channels
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int l16 = lane & 15, q4 = lane >> 4;
    const int head = b * g.H + h;
    const int c0 = seg * g.seg_chunks, t_begin = c0 * kChunk;
    const int t_end = g.T - t_begin < g.seg_chunks * kChunk ? g.T : t_begin + g.seg_chunks * kChunk;
    const int live = stream_tokens(g.lens, b, g.T);
    const int n_tok = live < t_begin ? 0 : (live < t_end ? live : t_end) - t_begin;
    const size_t row0 = (size_t)b * g.T + t_begin;

    // state: column m = 16 wave + l16; S[2s], S[2s + 1] hold rows 32 s + 8 q4 + r and
    // + 4, so that the pair is the operand of k-step s
    kr_float4 S[2 * KS];
    const int m = 16 * wave + l16;
    const size_t state_at = (size_t)(8 * q4) * D + m, slot = ((size_t)seg * heads + head) * D * D + state_at;
    const float* s_in = g.segments > 1 ? g.starts + slot : g.state + (size_t)head * D * D + state_at;
    #pragma unroll
    for (int s = 0; s < KS; s++)
        #pragma unroll
        for (int e = 0; e < 8; e++)
            S[2 * s + e / 4][e % 4] = MODE != SUMS ? s_in[(size_t)(32 * s + e) * D]
                                                   : map && 32 * s + 8 * q4 + e == m ? 1.0f : 0.0f;

    // what a thread stages: 8 channels of tokens 2p, 2p + 1
    const int ng = tid % (D / 8), p = tid / (D / 8);
    kr_half8 qq[2], kk[2], vv[2];
    const size_t first = row0 + 2 * p;
    const kr_half* qp = g.q + first * g.ldq + h * D + 8 * ng;
    const kr_half* kp = g.k + first * g.ldk + h * D + 8 * ng;
    const kr_half* vp = g.v + first * g.ldv + h * D + 8 * ng;
    const float* gp = g.gate + (row0 + lane) * g.ldg + h;
    const float* bp = g.beta + (row0 + lane) * g.ldb + h;
    float gate = 0.0f, beta = 0.0f;
    auto fetch = [&](int t0) {            // in order of t0
        #pragma unroll
        for (int e = 0; e < 2; e++) {
            const kr_half8 zero = {0, 0, 0, 0, 0, 0, 0, 0};
            qq[e] = kk[e] = vv[e] = zero;
            if (t0 + 2 * p + e < n_tok) {
                if (MODE == FORWARD) qq[e] = *reinterpret_cast<const kr_half8*>(qp + e * g.ldq);
                kk[e] = *reinterpret_cast<const kr_half8*>(kp + e * g.ldk);
                if (!map) vv[e] = *reinterpret_cast<const kr_half8*>(vp + e * g.ldv);
            }
        }
        qp += kChunk * g.ldq;
        kp += kChunk * g.ldk;
        vp += kChunk * g.ldv;
    };
    auto fetch_gates = [&](int t0) {
        const bool on = t0 + lane < n_tok;
        gate = on ? *gp : 0.0f;
        beta = on ? *bp : 0.0f;
        gp += kChunk * g.ldg;
        bp += kChunk * g.ldb;
    };
    kr_half* yp = g.y + (row0 + l16) * g.ldy + h * D + 16 * wave + 4 * q4;

    fetch(0);
    if (wave == 2) {
        fetch_gates(0);
        make_gates(sh.gates[0], gate, beta, lane);
        fetch_gates(kChunk);
    }
    for (int t0 = 0, c = 0; t0 < n_tok; t0 += kChunk, c++) {
        const int n = n_tok - t0 < kChunk ? n_tok - t0 : kChunk;
        #pragma unroll
        for (int e = 0; e < 2; e++) {
            if (MODE == FORWARD) sh.q[tok_unit<D>(2 * p + e, ng)] = qq[e];
            sh.k[tok_unit<D>(2 * p + e, ng)] = kk[e];
            sh.v[tok_unit<D>(2 * p + e, ng)] = vv[e];
        }
        const Gates& gates = sh.gates[c & 1];
        if (t0 + kChunk < n_tok) fetch(t0 + kChunk);
        if constexpr (MODE == STATES) {
            float* out = g.before + ((size_t)(c0 + c) * heads + head) * D * D + state_at;
            #pragma unroll
            for (int s = 0; s < KS; s++)
                #pragma unroll
                for (int e = 0; e < 8; e++) out[(size_t)(32 * s + e) * D] = S[2 * s + e / 4][e % 4];
        }
        __syncthreads();
        make_pairs<D, false, MODE == FORWARD>(sh.pairs, sh.q, sh.k, gates, wave, lane, [&]() {
            if (t0 + kChunk >= n_tok) return;
            make_gates(sh.gates[(c + 1) & 1], gate, beta, lane);
            fetch_gates(t0 + 2 * kChunk);
        });

        // the state's parts, with a scale for each column
        phase();
        const int ln = fresh(lane), l16 = ln & 15, q4 = ln >> 4;
        float big = 0.0f, up, down;
        #pragma unroll
        for (int s = 0; s < 2 * KS; s++)
            #pragma unroll
            for (int r = 0; r < 4; r++) big = fmaxf(big, fabsf(S[s][r]));
        power_scale(max_of_quarters(big), up, down);
        Parts8 sp[KS];
        #pragma unroll
        for (int s = 0; s < KS; s++)
            #pragma unroll
            for (int e = 0; e < 8; e++) {
                kr_half x, y;
                two_parts(S[2 * s + e / 4][e % 4], up, x, y);
                sp[s].hi[e] = x;
                sp[s].lo[e] = y;
            }

        phase();
        // X = v - e^a k S, rows t = 32 s + 8 q4 + e, column m; q S, rows m, columns i
        float X[2][8];
        kr_float4 from_s[4];
        if constexpr (MODE == FORWARD)
            #pragma unroll
            for (int it = 0; it < 4; it++) {
                from_s[it] = kr_float4{0, 0, 0, 0};
                #pragma unroll
                for (int s = 0; s < KS; s++) {
                    const kr_half8 x = sh.q[tok_unit<D>(16 * it + l16, 4 * s + q4)];
                    from_s[it] = mfma(sp[s].hi, x, from_s[it]);
                    from_s[it] = mfma(sp[s].lo, x, from_s[it]);
                }
            }
        #pragma unroll
        for (int s = 0; s < 2; s++) {
            const kr_half8 vc = channels16<D>(sh.v, s, wave, ln);
            #pragma unroll
            for (int hf = 0; hf < 2; hf++) {
                const int t = 32 * s + 8 * (l16 >> 2) + 4 * hf + (l16 & 3);
                kr_float4 z = {0, 0, 0, 0};
                #pragma unroll
                for (int kst = 0; kst < KS; kst++) {
                    const kr_half8 x = sh.k[tok_unit<D>(t, 4 * kst + q4)];
                    z = mfma(x, sp[kst].hi, z);
                    z = mfma(x, sp[kst].lo, z);
                }
                const kr_float4 e0 = *reinterpret_cast<const kr_float4*>(gates.e0 + 32 * s + 8 * q4 + 4 * hf);
                #pragma unroll
                for (int r = 0; r < 4; r++) X[s][4 * hf + r] = __builtin_fmaf(-(e0[r] * down), z[r], (float)vc[4 * hf + r]);
            }
        }
        phase();
        // u of the first half, then of the second; first all operands that they take
        Parts8 up8[2], n_of[2][2], a_of[2];
        float u_down[2], U[2][8], bt[2][8];
        kr_float4 n_f[2][2], a_f[2];
        #pragma unroll
        for (int s = 0; s < 2; s++)
            #pragma unroll
            for (int hf = 0; hf < 2; hf++) {
                const int t = 32 * s + 8 * (l16 >> 2) + 4 * hf + (l16 & 3), at = pair_unit(t, 4 * s + q4);
                n_of[s][hf] = Parts8{sh.pairs.mh[at], sh.pairs.ml[at]};
                n_f[s][hf] = *reinterpret_cast<const kr_float4*>(sh.pairs.n_down + 32 * s + 8 * q4 + 4 * hf);
                const kr_float4 b4 = *reinterpret_cast<const kr_float4*>(gates.beta + 32 * s + 8 * q4 + 4 * hf);
                #pragma unroll
                for (int r = 0; r < 4; r++) bt[s][4 * hf + r] = b4[r];
                if (s == 1) {
                    const int below = pair_unit(t, q4);
                    a_of[hf] = Parts8{sh.pairs.mh[below], sh.pairs.ml[below]};
                    a_f[hf] = *reinterpret_cast<const kr_float4*>(sh.pairs.a_down + 32 + 8 * q4 + 4 * hf);
                }
            }
        #pragma unroll
        for (int s = 0; s < 2; s++) {
            float x[8], x_down;
            if (s == 1) {
                #pragma unroll
                for (int hf = 0; hf < 2; hf++) {
                    const kr_float4 z = mfma3(a_of[hf].hi, a_of[hf].lo, up8[0], kr_float4{0, 0, 0, 0});
                    #pragma unroll
                    for (int r = 0; r < 4; r++) X[1][4 * hf + r] = __builtin_fmaf(-(a_f[hf][r] * u_down[0]), z[r], X[1][4 * hf + r]);
                }
            }
            #pragma unroll
            for (int e = 0; e < 8; e++) x[e] = bt[s][e] * X[s][e];
            const Parts8 xp = scaled8(x, x_down);
            #pragma unroll
            for (int hf = 0; hf < 2; hf++) {
                const kr_float4 z = mfma3(n_of[s][hf].hi, n_of[s][hf].lo, xp, kr_float4{0, 0, 0, 0});
                #pragma unroll
                for (int r = 0; r < 4; r++) X[s][4 * hf + r] = __builtin_fmaf(-(n_f[s][hf][r] * x_down), z[r], X[s][4 * hf + r]);
            }
            #pragma unroll
            for (int e = 0; e < 8; e++) U[s][e] = bt[s][e] * X[s][e];
            up8[s] = scaled8(U[s], u_down[s]);
        }
        phase();
        if constexpr (MODE == STATES) {
            float* out = g.diff + (((size_t)(c0 + c) * heads + head) * kChunk + 8 * q4) * D + m;
            #pragma unroll
            for (int s = 0; s < 2; s++)
                #pragma unroll
                for (int e = 0; e < 8; e++) out[(size_t)(32 * s + e) * D] = X[s][e];
        }
        if constexpr (MODE == FORWARD) {
            // y': rows m, columns i
            kr_float4 down_m, u0_m, u1_m;      // of the rows m that this lane has of y'
            #pragma unroll
            for (int r = 0; r < 4; r++) {
                down_m[r] = __shfl(down, 4 * q4 + r);
                u0_m[r] = __shfl(u_down[0], 4 * q4 + r);
                u1_m[r] = __shfl(u_down[1], 4 * q4 + r);
            }
            #pragma unroll
            for (int it = 0; it < 4; it++) {
                if (it == 2) phase();
                const int i = 16 * it + l16;
                kr_float4 in0 = {0, 0, 0, 0}, in1 = {0, 0, 0, 0};
                const int at = pair_unit(i, q4);
                in0 = mfma(up8[0].lo, sh.pairs.ph[at], in0);
                in0 = mfma(up8[0].hi, sh.pairs.pl[at], in0);
                in0 = mfma(up8[0].hi, sh.pairs.ph[at], in0);
                if (it >= 2) {
                    const int at1 = pair_unit(i, 4 + q4);
                    in1 = mfma(up8[1].lo, sh.pairs.ph[at1], in1);
                    in1 = mfma(up8[1].hi, sh.pairs.pl[at1], in1);
                    in1 = mfma(up8[1].hi, sh.pairs.ph[at1], in1);
                }
                const float pd = sh.pairs.p_down[i], e0 = gates.e0[i];
                kr_half4 y;
                #pragma unroll
                for (int r = 0; r < 4; r++) {
                    float x = from_s[it][r] * (down_m[r] * e0);
                    x = __builtin_fmaf(in0[r], pd * u0_m[r], x);
                    if (it >= 2) x = __builtin_fmaf(in1[r], pd * u1_m[r], x);
                    y[r] = kr_f16(x);
                }
                if (i < n) *reinterpret_cast<kr_half4*>(yp + 16 * it * g.ldy) = y;
            }
            yp += kChunk * g.ldy;
        }
        phase();
        // S <- e^a_end S + k' (e^(a_end - a) u)
        float x[2][8];
        #pragma unroll
        for (int s = 0; s < 2; s++)
            #pragma unroll
            for (int e = 0; e < 8; e++) x[s][e] = gates.e1[32 * s + 8 * q4 + e] * U[s][e];
        float x_up, x_down;
        power_scale(max_of_quarters(largest8(x[1], largest8(x[0]))), x_up, x_down);
        const Parts8 xp[2] = {parts8(x[0], x_up), parts8(x[1], x_up)};
        const float all = gates.all;
        #pragma unroll
        for (int st = 0; st < 2 * KS; st++) {
            kr_float4 add = {0, 0, 0, 0};
            #pragma unroll
            for (int s = 0; s < 2; s++) {
                const kr_half8 kc = channels_state<D>(sh.k, s, st, ln);
                add = mfma(kc, xp[s].lo, add);
                add = mfma(kc, xp[s].hi, add);
            }
            #pragma unroll
            for (int r = 0; r < 4; r++) S[st][r] = __builtin_fmaf(add[r], x_down, all * S[st][r]);
            if (st % 2) phase();
        }
        __syncthreads();
    }

    float* s_out = nullptr;
    if (MODE == SUMS) {
        s_out = (map ? g.maps : g.sums) + slot;
    } else if (MODE == FORWARD) {
        if (seg == g.segments - 1) s_out = g.state + (size_t)head * D * D + state_at;
    } else if ((live > t_begin || seg == 0) && live <= t_end) {       // the stream's end
        s_out = g.before + ((size_t)((live + kChunk - 1) / kChunk) * heads + head) * D * D + state_at;
    }
    if (s_out)
        #pragma unroll
        for (int s = 0; s < KS; s++)
            #pragma unroll
            for (int e = 0; e < 8; e++) s_out[(size_t)(32 * s + e) * D] = S[2 * s + e / 4][e % 4];
    if (MODE == FORWARD)
        for (long long i = (long long)n_tok * (D / 8) + tid; i < (long long)(t_end - t_begin) * (D / 8); i += 4 * D)
            *reinterpret_cast<kr_half8*>(g.y + (row0 + i / (D / 8)) * g.ldy + h * D + 8 * (i % (D / 8))) =
                kr_half8{0, 0, 0, 0, 0, 0, 0, 0};
}

template <int D>
__global__ void __launch_bounds__(4 * D, 2) delta_chunk_kernel(DeltaArgs g) {
    __shared__ DeltaShared<D> sh;
    int b = blockIdx.x / g.H;
    if (g.segments == 1) b = ranked_stream<4 * D>(g.lens, g.B, g.T, b, reinterpret_cast<int*>(&sh.pairs));
    walk_chunks<D, FORWARD>(g, sh, gridDim.x, b, blockIdx.x % g.H, blockIdx.y, false);
}

// ---------------------------------------------------------------------------
// Backward. With D the gradient of the state behind a chunk, from the last chunk to
// the first and again a wave for each 16 columns:
//   du = P' dy + e^(a_end - a) k D;   w = du - A' dX with dX = beta w (solved as r is,
//   with the transposed N and the halves in the other order);
//   D <- e^a_end D + (e^a q)' dy - (e^a k)' dX.
// It leaves D behind each chunk and w, from which, with the states and r of a forward
// pass, all chunks at once get the rest:
//   dv = dX;  dbeta = w r;  MP_ij = e^(a_i - a_j) dy_i u_j' (j <= i);
//   MA_ij = -e^(a_i - a_j) dX_i u_j' (j < i);  dq = e^a dy S' + MP k;
//   dk of the reading key = -e^a dX S' + MA k;
//   dk of the writing key = MP' q + MA' k + e^(a_end - a) u D';
//   da = q dq + k dk_read - k dk_write, and at the chunk's end sum D S_behind;
//   dg_i = sum of da from i to the chunk's end.
// ---------------------------------------------------------------------------
struct BackArgs {
    const kr_half* q;
    const kr_half* k;
    const kr_half* dy;
    long long ldq, ldk, ldy;
    const float* gate;
    const float* beta;
    long long ldg, ldb;
    const int32_t* lens;
    const float* dstate;          // null: zeros
    float* dstate0;
    float* behind;                // [chunks][heads][D][D]
    float* w;                     // [chunks][heads][64][D]
    const float* before;          // of the forward pass: states, r
    const float* diff;
    kr_half* dq;                  // [B, T, H, D]
    kr_half* dk;
    kr_half* dv;
    float* dgate;                 // [B, T, H]
    float* dbeta;
    float* sums;                  // [segments][heads][D][D], what a segment adds to D
    float* ends;                  // [segments][heads][D][D], D behind the segments (time split)
    int B, T, H;
    int seg_chunks, segments;
};

// SUM: only what a segment adds to D, from zero behind it.
template <int D, bool SUM>
__device__ __forceinline__ void walk_back(const BackArgs& g, DeltaShared<D>& sh, int heads, int b, int h, int seg) {
    constexpr int KS = D / 32;            // dy is in v's place
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int l16 = lane & 15, q4 = lane >> 4;
    const int head = b * g.H + h;
    const int c0 = seg * g.seg_chunks, t_begin = c0 * kChunk;
    const int t_end = g.T - t_begin < g.seg_chunks * kChunk ? g.T : t_begin + g.seg_chunks * kChunk;
    const int live = stream_tokens(g.lens, b, g.T);
    const int n_tok = live < t_begin ? 0 : (live < t_end ? live : t_end) - t_begin;
    const int chunks = (n_tok + kChunk - 1) / kChunk;
    const size_t row0 = (size_t)b * g.T + t_begin;

    kr_float4 S[2 * KS];                  // D, laid out as the forward pass's state
    const int m = 16 * wave + l16;
    const size_t state_at = (size_t)(8 * q4) * D + m, slot = ((size_t)seg * heads + head) * D * D + state_at;
    const float* d_in = SUM ? nullptr : g.segments > 1 ? g.ends + slot
                        : g.dstate ? g.dstate + (size_t)head * D * D + state_at : nullptr;
    #pragma unroll
    for (int s = 0; s < KS; s++)
        #pragma unroll
        for (int e = 0; e < 8; e++) S[2 * s + e / 4][e % 4] = d_in ? d_in[(size_t)(32 * s + e) * D] : 0.0f;

    const int ng = tid % (D / 8), p = tid / (D / 8);
    kr_half8 qq[2], kk[2], vv[2];
    auto fetch = [&](int t0) {
        #pragma unroll
        for (int e = 0; e < 2; e++) {
            const kr_half8 zero = {0, 0, 0, 0, 0, 0, 0, 0};
            qq[e] = kk[e] = vv[e] = zero;
            const int t = t0 + 2 * p + e;
            if (t < n_tok) {
                const size_t row = row0 + t;
                qq[e] = *reinterpret_cast<const kr_half8*>(g.q + row * g.ldq + h * D + 8 * ng);
                kk[e] = *reinterpret_cast<const kr_half8*>(g.k + row * g.ldk + h * D + 8 * ng);
                vv[e] = *reinterpret_cast<const kr_half8*>(g.dy + row * g.ldy + h * D + 8 * ng);
            }
        }
    };
    float gate = 0.0f, beta = 0.0f;
    auto fetch_gates = [&](int t0) {
        const bool on = t0 >= 0 && t0 + lane < n_tok;
        gate = on ? g.gate[(row0 + t0 + lane) * g.ldg + h] : 0.0f;
        beta = on ? g.beta[(row0 + t0 + lane) * g.ldb + h] : 0.0f;
    };
    if (chunks > 0) {
        fetch((chunks - 1) * kChunk);
        if (wave == 2) {
            fetch_gates((chunks - 1) * kChunk);
            make_gates(sh.gates[(chunks - 1) & 1], gate, beta, lane);
            fetch_gates((chunks - 2) * kChunk);
        }
    }
    for (int c = chunks - 1; c >= 0; c--) {
        #pragma unroll
        for (int e = 0; e < 2; e++) {
            sh.q[tok_unit<D>(2 * p + e, ng)] = qq[e];
            sh.k[tok_unit<D>(2 * p + e, ng)] = kk[e];
            sh.v[tok_unit<D>(2 * p + e, ng)] = vv[e];
        }
        const Gates& gates = sh.gates[c & 1];
        if (c > 0) fetch((c - 1) * kChunk);
        if constexpr (!SUM) {
            float* out = g.behind + ((size_t)(c0 + c) * heads + head) * D * D + state_at;
            #pragma unroll
            for (int s = 0; s < KS; s++)
                #pragma unroll
                for (int e = 0; e < 8; e++) out[(size_t)(32 * s + e) * D] = S[2 * s + e / 4][e % 4];
        }
        __syncthreads();
        make_pairs<D, true, true>(sh.pairs, sh.q, sh.k, gates, wave, lane, [&]() {
            if (c == 0) return;
            make_gates(sh.gates[(c - 1) & 1], gate, beta, lane);
            fetch_gates((c - 2) * kChunk);
        });
        phase();
        const int ln = fresh(lane), l16 = ln & 15, q4 = ln >> 4;
        float big = 0.0f, up, down;
        #pragma unroll
        for (int s = 0; s < 2 * KS; s++)
            #pragma unroll
            for (int r = 0; r < 4; r++) big = fmaxf(big, fabsf(S[s][r]));
        power_scale(max_of_quarters(big), up, down);
        Parts8 sp[KS];
        #pragma unroll
        for (int s = 0; s < KS; s++)
            #pragma unroll
            for (int e = 0; e < 8; e++) {
                kr_half x, y;
                two_parts(S[2 * s + e / 4][e % 4], up, x, y);
                sp[s].hi[e] = x;
                sp[s].lo[e] = y;
            }
        phase();
        // du, rows t = 32 s + 8 q4 + e, column m
        float X[2][8];
        const kr_half8 dyc[2] = {channels16<D>(sh.v, 0, wave, ln), channels16<D>(sh.v, 1, wave, ln)};
        #pragma unroll
        for (int s = 0; s < 2; s++)
            #pragma unroll
            for (int hf = 0; hf < 2; hf++) {
                const int t = 32 * s + 8 * (l16 >> 2) + 4 * hf + (l16 & 3);
                kr_float4 z = {0, 0, 0, 0}, in = {0, 0, 0, 0};
                #pragma unroll
                for (int kst = 0; kst < KS; kst++) {
                    const kr_half8 x = sh.k[tok_unit<D>(t, 4 * kst + q4)];
                    z = mfma(x, sp[kst].lo, z);
                    z = mfma(x, sp[kst].hi, z);
                }
                #pragma unroll
                for (int is = s; is < 2; is++) {
                    const int at = pair_unit(t, 4 * is + q4);
                    in = mfma(sh.pairs.pl[at], dyc[is], in);
                    in = mfma(sh.pairs.ph[at], dyc[is], in);
                }
                const kr_float4 e1 = *reinterpret_cast<const kr_float4*>(gates.e1 + 32 * s + 8 * q4 + 4 * hf);
                const kr_float4 f = *reinterpret_cast<const kr_float4*>(sh.pairs.p_down + 32 * s + 8 * q4 + 4 * hf);
                #pragma unroll
                for (int r = 0; r < 4; r++) X[s][4 * hf + r] = __builtin_fmaf(e1[r] * down, z[r], f[r] * in[r]);
            }
        phase();
        // w of the second half, then of the first; first all operands that they take
        Parts8 dx1, n_of[2][2], a_of[2];
        float dx1_down = 0.0f, dX[2][8], bt[2][8];
        kr_float4 n_f[2][2], a_f[2];
        #pragma unroll
        for (int s = 0; s < 2; s++)
            #pragma unroll
            for (int hf = 0; hf < 2; hf++) {
                const int t = 32 * s + 8 * (l16 >> 2) + 4 * hf + (l16 & 3), at = pair_unit(t, 4 * s + q4);
                n_of[s][hf] = Parts8{sh.pairs.mh[at], sh.pairs.ml[at]};
                n_f[s][hf] = *reinterpret_cast<const kr_float4*>(sh.pairs.n_down + 32 * s + 8 * q4 + 4 * hf);
                const kr_float4 b4 = *reinterpret_cast<const kr_float4*>(gates.beta + 32 * s + 8 * q4 + 4 * hf);
                #pragma unroll
                for (int r = 0; r < 4; r++) bt[s][4 * hf + r] = b4[r];
                if (s == 0) {
                    const int above = pair_unit(t, 4 + q4);
                    a_of[hf] = Parts8{sh.pairs.mh[above], sh.pairs.ml[above]};
                    a_f[hf] = *reinterpret_cast<const kr_float4*>(sh.pairs.a_down + 8 * q4 + 4 * hf);
                }
            }
        #pragma unroll
        for (int s = 1; s >= 0; s--) {
            float x[8], x_down;
            if (s == 0) {
                #pragma unroll
                for (int hf = 0; hf < 2; hf++) {
                    const kr_float4 z = mfma3(a_of[hf].hi, a_of[hf].lo, dx1, kr_float4{0, 0, 0, 0});
                    #pragma unroll
                    for (int r = 0; r < 4; r++) X[0][4 * hf + r] = __builtin_fmaf(-(a_f[hf][r] * dx1_down), z[r], X[0][4 * hf + r]);
                }
            }
            #pragma unroll
            for (int e = 0; e < 8; e++) x[e] = bt[s][e] * X[s][e];
            const Parts8 xp = scaled8(x, x_down);
            #pragma unroll
            for (int hf = 0; hf < 2; hf++) {
                const kr_float4 z = mfma3(n_of[s][hf].hi, n_of[s][hf].lo, xp, kr_float4{0, 0, 0, 0});
                #pragma unroll
                for (int r = 0; r < 4; r++) X[s][4 * hf + r] = __builtin_fmaf(-(n_f[s][hf][r] * x_down), z[r], X[s][4 * hf + r]);
            }
            #pragma unroll
            for (int e = 0; e < 8; e++) dX[s][e] = bt[s][e] * X[s][e];
            if (s == 1) dx1 = scaled8(dX[1], dx1_down);
        }
        if constexpr (!SUM) {
            float* out = g.w + (((size_t)(c0 + c) * heads + head) * kChunk + 8 * q4) * D + m;
            #pragma unroll
            for (int s = 0; s < 2; s++)
                #pragma unroll
                for (int e = 0; e < 8; e++) out[(size_t)(32 * s + e) * D] = X[s][e];
        }
        phase();
        // D <- e^a_end D + q' (e^a dy) - k' (e^a dX)
        float yx[2][8];
        #pragma unroll
        for (int s = 0; s < 2; s++)
            #pragma unroll
            for (int e = 0; e < 8; e++) {
                const float e0 = gates.e0[32 * s + 8 * q4 + e];
                yx[s][e] = e0 * (float)dyc[s][e];
                dX[s][e] *= -e0;
            }
        float y_up, y_down, x_up, x_down;
        power_scale(max_of_quarters(largest8(yx[1], largest8(yx[0]))), y_up, y_down);
        power_scale(max_of_quarters(largest8(dX[1], largest8(dX[0]))), x_up, x_down);
        const Parts8 yp[2] = {parts8(yx[0], y_up), parts8(yx[1], y_up)};
        const Parts8 xp[2] = {parts8(dX[0], x_up), parts8(dX[1], x_up)};
        const float all = gates.all;
        #pragma unroll
        for (int st = 0; st < 2 * KS; st++) {
            kr_float4 from_y = {0, 0, 0, 0}, from_x = {0, 0, 0, 0};
            #pragma unroll
            for (int s = 0; s < 2; s++) {
                const kr_half8 qc = channels_state<D>(sh.q, s, st, ln), kc = channels_state<D>(sh.k, s, st, ln);
                from_y = mfma(qc, yp[s].lo, from_y);
                from_y = mfma(qc, yp[s].hi, from_y);
                from_x = mfma(kc, xp[s].lo, from_x);
                from_x = mfma(kc, xp[s].hi, from_x);
            }
            #pragma unroll
            for (int r = 0; r < 4; r++)
                S[st][r] = __builtin_fmaf(from_x[r], x_down, __builtin_fmaf(from_y[r], y_down, all * S[st][r]));
            if (st % 2) phase();
        }
        __syncthreads();
    }
    float* out = SUM ? g.sums + slot : seg == 0 ? g.dstate0 + (size_t)head * D * D + state_at : nullptr;
    if (out)
        #pragma unroll
        for (int s = 0; s < KS; s++)
            #pragma unroll
            for (int e = 0; e < 8; e++) out[(size_t)(32 * s + e) * D] = S[2 * s + e / 4][e % 4];
}

// The states of a forward pass and D, one beside the other.
template <int D>
__global__ void __launch_bounds__(4 * D, 2) delta_both_kernel(DeltaArgs f, BackArgs g) {
    __shared__ DeltaShared<D> sh;
    int b = blockIdx.x / g.H;
    if (g.segments == 1) b = ranked_stream<4 * D>(g.lens, g.B, g.T, b, reinterpret_cast<int*>(&sh.pairs));
    if (blockIdx.z == 0) walk_chunks<D, STATES>(f, sh, gridDim.x, b, blockIdx.x % g.H, blockIdx.y, false);
    else walk_back<D, false>(g, sh, gridDim.x, b, blockIdx.x % g.H, blockIdx.y);
}

// ---------------------------------------------------------------------------
// Time split, for few heads: what each segment makes of a state, S -> map S + sum, is
// computed for all segments at once, the states at their starts follow one from
// the other, and then all segments run. Backward, D -> map' D + sum.
// z of the sums' launch: 0 sums, 1 maps, 2 D's sums; of the states': 0 forward, 1 back.
// Three times the work, side by side: 1 x 1777 x 8 heads of 128 274 -> 77 us (14 segments:
// sums 19, join 36, walk 24), gradients of 1 x 2000 x 12 of 64 394 -> 83 (28, 12, 28, and
// 21 for the chunks' gradients).
// ---------------------------------------------------------------------------
template <int D>
__global__ void __launch_bounds__(4 * D, 2) delta_sums_kernel(DeltaArgs f, BackArgs g) {
    __shared__ DeltaShared<D> sh;
    const int seg = blockIdx.y, b = blockIdx.x / f.H, h = blockIdx.x % f.H;
    if (blockIdx.z < 2) {
        if (blockIdx.z == 0 && seg == f.segments - 1) return;         // not needed
        walk_chunks<D, SUMS>(f, sh, gridDim.x, b, h, seg, blockIdx.z == 1);
    } else if (seg > 0) {
        walk_back<D, true>(g, sh, gridDim.x, b, h, seg);
    }
}

// 16 columns of a head: a wave has 16 rows of every segment's map, read two segments
// ahead (or every step waits for memory); the column passes through LDS, [m][n] in two
// buffers, with a barrier a step that uses them: a stream's segments with tokens follow
// one another, and steps of those without touch neither. Bound by a step's chain: 1.2 us
// for D = 64, 2.9 for 128 (values taken apart by 8 waves on one CU, a barrier, 12 products).
template <int D>
struct JoinPiece {
    float map[D / 32][8], sum[4];
};
template <int D, bool BACK>
__device__ __forceinline__ void join_segments(const DeltaArgs& f, const float* sums, const float* first, float* out,
                                              float (&S)[2][16 * (D + 4)], int heads, int head, int m0) {
    constexpr int KS = D / 32, LD = D + 4;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int l16 = lane & 15, q4 = lane >> 4, m = m0 + l16;
    const int n = f.segments, rows = 16 * wave, live = stream_tokens(f.lens, head / f.H, f.T);
    const size_t step = (size_t)heads * D * D, at = (size_t)head * D * D;
    const int sum_at = (rows + 4 * q4) * D + m;           // of 4 rows in a column
    const int map_at = BACK ? 8 * q4 * D + rows + l16 : (rows + l16) * D + 8 * q4;
    // step i takes segment seg(i)'s map and sum, and gives the next one's start (or end)
    auto seg = [&](int i) { return BACK ? n - 1 - i : i; };
    auto fetch = [&](int i, JoinPiece<D>& o) {            // without a branch, so that waits are counted
        i = i < n - 2 ? i : n - 2;
        const float* p = f.maps + at + seg(i) * step + map_at;
        #pragma unroll
        for (int s = 0; s < KS; s++)
            #pragma unroll
            for (int e = 0; e < 8; e++)
                o.map[s][e] = BACK ? p[(32 * s + e) * D] : reinterpret_cast<const kr_float4*>(p + 32 * s)[e / 4][e % 4];
        #pragma unroll
        for (int r = 0; r < 4; r++) o.sum[r] = sums[at + seg(i) * step + sum_at + r * D];
    };
    kr_float4 x;
    #pragma unroll
    for (int r = 0; r < 4; r++) x[r] = first ? first[at + sum_at + r * D] : 0.0f;
    auto take = [&](int i, JoinPiece<D>& o) {
        float* to = out + at + seg(i) * step + sum_at;
        #pragma unroll
        for (int r = 0; r < 4; r++) to[r * D] = x[r];
        // no token: x stays, and so does LDS, which slower waves may still read
        const bool tokens = seg(i) * f.seg_chunks * kChunk < live;
        float* col = S[i & 1];
        if (tokens) *reinterpret_cast<kr_float4*>(col + l16 * LD + rows + 4 * q4) = x;
        // the map's parts, with a scale for each row
        Parts8 mp[KS];
        float big = 0.0f, up, m_down, x_down;
        #pragma unroll
        for (int s = 0; s < KS; s++) big = largest8(o.map[s], big);
        power_scale(max_of_quarters(big), up, m_down);
        #pragma unroll
        for (int s = 0; s < KS; s++) mp[s] = parts8(o.map[s], up);
        const kr_float4 add = {o.sum[0], o.sum[1], o.sum[2], o.sum[3]};
        fetch(i + 2, o);
        if (!tokens) return;
        __syncthreads();
        float c[KS][8];
        big = 0.0f;
        #pragma unroll
        for (int s = 0; s < KS; s++) {
            const kr_float4* p = reinterpret_cast<const kr_float4*>(col + l16 * LD + 32 * s + 8 * q4);
            #pragma unroll
            for (int e = 0; e < 8; e++) c[s][e] = p[e / 4][e % 4];
            big = largest8(c[s], big);
        }
        power_scale(max_of_quarters(big), up, x_down);
        kr_float4 z = {0, 0, 0, 0};
        #pragma unroll
        for (int s = 0; s < KS; s++) z = mfma3(mp[s].hi, mp[s].lo, parts8(c[s], up), z);
        #pragma unroll
        for (int r = 0; r < 4; r++) x[r] = __builtin_fmaf(z[r], x_down * __shfl(m_down, 4 * q4 + r), add[r]);
    };
    JoinPiece<D> a, b;
    fetch(0, a);
    fetch(1, b);
    int i = 0;
    for (; i + 2 < n; i += 2) {
        take(i, a);
        take(i + 1, b);
    }
    if (i < n - 1) take(i, a);
    float* to = out + at + seg(n - 1) * step + sum_at;
    #pragma unroll
    for (int r = 0; r < 4; r++) to[r * D] = x[r];
}

template <int D>
__global__ void __launch_bounds__(4 * D) delta_join_kernel(DeltaArgs f, BackArgs g) {
    __shared__ __attribute__((aligned(16))) float S[2][16 * (D + 4)];
    const int heads = gridDim.x, head = blockIdx.x, m0 = 16 * blockIdx.y;
    if (blockIdx.z == 0) join_segments<D, false>(f, f.sums, f.state, f.starts, S, heads, head, m0);
    else join_segments<D, true>(f, g.sums, g.dstate, g.ends, S, heads, head, m0);
}

// A workgroup of 4 waves for each head and chunk, a wave for 16 tokens, as those that
// read and as those that write. 64 rows of S, then of D, are in LDS at a time.
// Bound: waits for memory with 8 waves a CU (77 KB of LDS a workgroup): a chunk's 130 KB
// are loaded, then computed on. Measured on MI355X, 48 streams of 256..1024 x 12 heads of
// 64: 278 us (0.55 GB, 2 TB/s; VALU 38% busy), the walks before it 243 (0.53 GB). Eight waves
// a workgroup, four for each side, spill at 128 registers: 634.
template <int D>
struct GradShared {
    kr_half8 q[kChunk * D / 8], k[kChunk * D / 8], dy[kChunk * D / 8];             // by tokens
    kr_half8 uh[kChunk * D / 8], ul[kChunk * D / 8], xh[kChunk * D / 8], xl[kChunk * D / 8];   // u, dX
    kr_half8 sh[kChunk * D / 8], sl[kChunk * D / 8];                               // 64 rows of S or D
    float u_down[kChunk], x_down[kChunk], s_down[kChunk], da[kChunk], dot[4];
    Gates gates;
};

// 8 values of a row that D / 8 neighbouring lanes hold, in two parts.
template <int D>
__device__ __forceinline__ Parts8 row_parts(const float (&x)[8], float& down) {
    float big = largest8(x), up;
    big = fmaxf(big, kr_xor<1>(big));
    big = fmaxf(big, kr_xor<2>(big));
    big = fmaxf(big, kr_xor<4>(big));
    if (D == 128) big = fmaxf(big, kr_xor<8>(big));
    power_scale(big, up, down);
    return parts8(x, up);
}

template <int D>
__device__ __forceinline__ float row_sum(float x) {
    x += kr_xor<1>(x);
    x += kr_xor<2>(x);
    x += kr_xor<4>(x);
    if (D == 128) x += kr_xor<8>(x);
    return x;
}

template <int D>
__global__ void __launch_bounds__(256, D == 64 ? 2 : 1) delta_grad_kernel(BackArgs g) {
    constexpr int KS = D / 32, UNITS = D / 8, PASSES = kChunk * UNITS / 256;
    __shared__ GradShared<D> sh;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int l16 = lane & 15, q4 = lane >> 4;
    const int heads = gridDim.x, head = blockIdx.x, c = blockIdx.y, b = head / g.H, h = head % g.H;
    const int t0 = c * kChunk;
    const int live = stream_tokens(g.lens, b, g.T) - t0, n = live < 0 ? 0 : live < kChunk ? live : kChunk;
    const int rows = g.T - t0 < kChunk ? g.T - t0 : kChunk;
    const size_t row0 = (size_t)b * g.T + t0;
    const long long ldo = (long long)g.H * D;
    const int unit = tid % UNITS, first = tid / UNITS;     // 8 channels of tokens first + 256 / UNITS i
    if (n == 0) {
        const kr_half8 zero = {0, 0, 0, 0, 0, 0, 0, 0};
        for (int t = first; t < rows; t += 256 / UNITS) {
            const size_t o = (row0 + t) * ldo + h * D + 8 * unit;
            *reinterpret_cast<kr_half8*>(g.dq + o) = zero;
            *reinterpret_cast<kr_half8*>(g.dk + o) = zero;
            *reinterpret_cast<kr_half8*>(g.dv + o) = zero;
        }
        if (tid < rows) g.dgate[(row0 + tid) * g.H + h] = g.dbeta[(row0 + tid) * g.H + h] = 0.0f;
        return;
    }
    if (wave == 0) {
        const bool on = lane < n;
        make_gates(sh.gates, on ? g.gate[(row0 + lane) * g.ldg + h] : 0.0f,
                   on ? g.beta[(row0 + lane) * g.ldb + h] : 0.0f, lane);
    }
    const size_t diff_at = ((size_t)c * heads + head) * kChunk * D;
    #pragma unroll
    for (int i = 0; i < PASSES; i++) {
        const int t = first + 256 / UNITS * i;
        const bool on = t < n;
        const kr_half8 zero = {0, 0, 0, 0, 0, 0, 0, 0};
        kr_half8 x = zero, y = zero, z = zero;
        float beta = 0.0f;
        if (on) {
            x = *reinterpret_cast<const kr_half8*>(g.q + (row0 + t) * g.ldq + h * D + 8 * unit);
            y = *reinterpret_cast<const kr_half8*>(g.k + (row0 + t) * g.ldk + h * D + 8 * unit);
            z = *reinterpret_cast<const kr_half8*>(g.dy + (row0 + t) * g.ldy + h * D + 8 * unit);
            beta = g.beta[(row0 + t) * g.ldb + h];
        }
        const int at = tok_unit<D>(t, unit);
        sh.q[at] = x;
        sh.k[at] = y;
        sh.dy[at] = z;
        float r[8], w[8], dot = 0.0f;
        const kr_float4* rp = reinterpret_cast<const kr_float4*>(g.diff + diff_at + (size_t)t * D + 8 * unit);
        const kr_float4* wp = reinterpret_cast<const kr_float4*>(g.w + diff_at + (size_t)t * D + 8 * unit);
        kr_half8 dv;
        #pragma unroll
        for (int e = 0; e < 8; e++) {
            r[e] = rp[e / 4][e % 4];
            w[e] = wp[e / 4][e % 4];
            dot = __builtin_fmaf(r[e], w[e], dot);
            r[e] *= beta;
            w[e] *= beta;
            dv[e] = kr_f16(w[e]);
        }
        float down;
        const Parts8 up = row_parts<D>(r, down);
        sh.uh[at] = up.hi;
        sh.ul[at] = up.lo;
        if (unit == 0) sh.u_down[t] = down;
        const Parts8 xp = row_parts<D>(w, down);
        sh.xh[at] = xp.hi;
        sh.xl[at] = xp.lo;
        dot = row_sum<D>(dot);
        if (unit == 0) sh.x_down[t] = down;
        if (t < rows) {
            *reinterpret_cast<kr_half8*>(g.dv + (row0 + t) * ldo + h * D + 8 * unit) = on ? dv : zero;
            if (unit == 0) g.dbeta[(row0 + t) * g.H + h] = on ? dot : 0.0f;
        }
    }
    float dot = 0.0f;                     // sum D S_behind
    auto stage = [&](const float* from, const float* times, int nb) {
        #pragma unroll
        for (int i = 0; i < PASSES; i++) {
            const int r = first + 256 / UNITS * i;
            const size_t at = (size_t)(64 * nb + r) * D + 8 * unit;
            const kr_float4* fp = reinterpret_cast<const kr_float4*>(from + at);
            float x[8], down;
            #pragma unroll
            for (int e = 0; e < 8; e++) x[e] = fp[e / 4][e % 4];
            if (times) {
                const kr_float4* tp = reinterpret_cast<const kr_float4*>(times + at);
                #pragma unroll
                for (int e = 0; e < 8; e++) dot = __builtin_fmaf(x[e], tp[e / 4][e % 4], dot);
            }
            const Parts8 p = row_parts<D>(x, down);
            sh.sh[tok_unit<D>(r, unit)] = p.hi;
            sh.sl[tok_unit<D>(r, unit)] = p.lo;
            if (unit == 0) sh.s_down[r] = down;
        }
    };
    const float* before = g.before + ((size_t)c * heads + head) * D * D;
    const float* after = before + (size_t)heads * D * D;
    const float* behind = g.behind + ((size_t)c * heads + head) * D * D;
    stage(before, nullptr, 0);
    __syncthreads();

    const int mine = 16 * wave + l16;     // this lane's token
    const double a = sh.gates.a[mine];
    const float e0 = sh.gates.e0[mine], e1 = sh.gates.e1[mine];
    const float u_mine = sh.u_down[mine], x_mine = sh.x_down[mine];
    // this lane's dy and dX as tokens that read, u as tokens that write
    kr_half8 yv[KS];
    Parts8 xv[KS], uv[KS];
    #pragma unroll
    for (int s = 0; s < KS; s++) {
        const int at = tok_unit<D>(mine, 4 * s + q4);
        yv[s] = sh.dy[at];
        xv[s] = Parts8{sh.xh[at], sh.xl[at]};
        uv[s] = Parts8{sh.uh[at], sh.ul[at]};
    }
    // rows of MP and MA (other tokens j = 32 s + 8 q4 + e), then columns (i = ..)
    Parts8 mp[2], ma[2], mpt[2], mat[2];
    float mp_down, ma_down, mpt_down, mat_down;
    {
        float P[2][8], A[2][8];
        #pragma unroll
        for (int s = 0; s < 2; s++)
            #pragma unroll
            for (int hf = 0; hf < 2; hf++) {
                kr_float4 zp = {0, 0, 0, 0}, za = {0, 0, 0, 0};
                const int t = 32 * s + 8 * (l16 >> 2) + 4 * hf + (l16 & 3);
                if (s <= wave / 2) {
                    #pragma unroll
                    for (int kst = 0; kst < KS; kst++) {
                        const int at = tok_unit<D>(t, 4 * kst + q4);
                        const kr_half8 uh = sh.uh[at], ul = sh.ul[at];
                        zp = mfma(ul, yv[kst], zp);
                        zp = mfma(uh, yv[kst], zp);
                        za = mfma3(uh, ul, xv[kst], za);
                    }
                }
                #pragma unroll
                for (int r = 0; r < 4; r++) {
                    const int j = 32 * s + 8 * q4 + 4 * hf + r;
                    const float f = sh.u_down[j] * __builtin_amdgcn_exp2f((float)(a - sh.gates.a[j]));
                    P[s][4 * hf + r] = j <= mine ? zp[r] * f : 0.0f;
                    A[s][4 * hf + r] = j < mine ? -(za[r] * x_mine) * f : 0.0f;
                }
            }
        float up;
        power_scale(max_of_quarters(largest8(P[1], largest8(P[0]))), up, mp_down);
        mp[0] = parts8(P[0], up);
        mp[1] = parts8(P[1], up);
        power_scale(max_of_quarters(largest8(A[1], largest8(A[0]))), up, ma_down);
        ma[0] = parts8(A[0], up);
        ma[1] = parts8(A[1], up);
        #pragma unroll
        for (int s = 0; s < 2; s++)
            #pragma unroll
            for (int hf = 0; hf < 2; hf++) {
                kr_float4 zp = {0, 0, 0, 0}, za = {0, 0, 0, 0};
                const int t = 32 * s + 8 * (l16 >> 2) + 4 * hf + (l16 & 3);
                if (s >= wave / 2) {
                    #pragma unroll
                    for (int kst = 0; kst < KS; kst++) {
                        const int at = tok_unit<D>(t, 4 * kst + q4);
                        const kr_half8 y = sh.dy[at];
                        zp = mfma(y, uv[kst].lo, zp);
                        zp = mfma(y, uv[kst].hi, zp);
                        za = mfma3(sh.xh[at], sh.xl[at], uv[kst], za);
                    }
                }
                #pragma unroll
                for (int r = 0; r < 4; r++) {
                    const int i = 32 * s + 8 * q4 + 4 * hf + r;
                    const float f = u_mine * __builtin_amdgcn_exp2f((float)(sh.gates.a[i] - a));
                    P[s][4 * hf + r] = i >= mine ? zp[r] * f : 0.0f;
                    A[s][4 * hf + r] = i > mine ? -(za[r] * sh.x_down[i]) * f : 0.0f;
                }
            }
        power_scale(max_of_quarters(largest8(P[1], largest8(P[0]))), up, mpt_down);
        mpt[0] = parts8(P[0], up);
        mpt[1] = parts8(P[1], up);
        power_scale(max_of_quarters(largest8(A[1], largest8(A[0]))), up, mat_down);
        mat[0] = parts8(A[0], up);
        mat[1] = parts8(A[1], up);
    }
    // 64 channels at a time: rows n of 16, this lane's token
    float da = 0.0f;
    for (int nb = 0; nb < D / 64; nb++) {
        if (nb > 0) {
            __syncthreads();
            stage(before, nullptr, nb);
            __syncthreads();
        }
        kr_float4 dq[4], read[4], write[4];
        #pragma unroll
        for (int nt = 0; nt < 4; nt++) {
            kr_float4 zq = {0, 0, 0, 0}, zk = {0, 0, 0, 0}, pk = {0, 0, 0, 0}, ak = {0, 0, 0, 0};
            #pragma unroll
            for (int s = 0; s < KS; s++) {
                const int at = tok_unit<D>(16 * nt + l16, 4 * s + q4);
                const kr_half8 hi = sh.sh[at], lo = sh.sl[at];
                zq = mfma(lo, yv[s], zq);
                zq = mfma(hi, yv[s], zq);
                zk = mfma3(hi, lo, xv[s], zk);
            }
            #pragma unroll
            for (int s = 0; s < 2; s++) {
                if (s > wave / 2) continue;
                const kr_half8 kc = channels16<D>(sh.k, s, 4 * nb + nt, lane);
                pk = mfma(kc, mp[s].lo, pk);
                pk = mfma(kc, mp[s].hi, pk);
                ak = mfma(kc, ma[s].lo, ak);
                ak = mfma(kc, ma[s].hi, ak);
            }
            const kr_float4 sd = *reinterpret_cast<const kr_float4*>(sh.s_down + 16 * nt + 4 * q4);
            #pragma unroll
            for (int r = 0; r < 4; r++) {
                dq[nt][r] = __builtin_fmaf(pk[r], mp_down, zq[r] * (sd[r] * e0));
                read[nt][r] = __builtin_fmaf(ak[r], ma_down, -(zk[r] * x_mine) * (sd[r] * e0));
            }
        }
        __syncthreads();
        stage(behind, after, nb);
        __syncthreads();
        #pragma unroll
        for (int nt = 0; nt < 4; nt++) {
            kr_float4 zu = {0, 0, 0, 0}, pq = {0, 0, 0, 0}, ak = {0, 0, 0, 0};
            #pragma unroll
            for (int s = 0; s < KS; s++) {
                const int at = tok_unit<D>(16 * nt + l16, 4 * s + q4);
                zu = mfma3(sh.sh[at], sh.sl[at], uv[s], zu);
            }
            #pragma unroll
            for (int s = 0; s < 2; s++) {
                if (s < wave / 2) continue;
                const kr_half8 qc = channels16<D>(sh.q, s, 4 * nb + nt, lane);
                const kr_half8 kc = channels16<D>(sh.k, s, 4 * nb + nt, lane);
                pq = mfma(qc, mpt[s].lo, pq);
                pq = mfma(qc, mpt[s].hi, pq);
                ak = mfma(kc, mat[s].lo, ak);
                ak = mfma(kc, mat[s].hi, ak);
            }
            const kr_float4 sd = *reinterpret_cast<const kr_float4*>(sh.s_down + 16 * nt + 4 * q4);
            #pragma unroll
            for (int r = 0; r < 4; r++)
                write[nt][r] = __builtin_fmaf(pq[r], mpt_down,
                                              __builtin_fmaf(ak[r], mat_down, (zu[r] * u_mine) * (sd[r] * e1)));
        }
        #pragma unroll
        for (int nt = 0; nt < 4; nt++) {
            const int ch = 64 * nb + 16 * nt + 4 * q4;
            const int at = tok_unit<D>(mine, ch / 8);
            const kr_half4 qv = reinterpret_cast<const kr_half4*>(sh.q + at)[ch / 4 & 1];
            const kr_half4 kv = reinterpret_cast<const kr_half4*>(sh.k + at)[ch / 4 & 1];
            kr_half4 oq, ok;
            #pragma unroll
            for (int r = 0; r < 4; r++) {
                da = __builtin_fmaf((float)qv[r], dq[nt][r], da);
                da = __builtin_fmaf((float)kv[r], read[nt][r] - write[nt][r], da);
                oq[r] = kr_f16(dq[nt][r]);
                ok[r] = kr_f16(read[nt][r] + write[nt][r]);
            }
            if (mine < rows) {
                const kr_half4 zero = {0, 0, 0, 0};
                const size_t o = (row0 + mine) * ldo + h * D + ch;
                *reinterpret_cast<kr_half4*>(g.dq + o) = mine < n ? oq : zero;
                *reinterpret_cast<kr_half4*>(g.dk + o) = mine < n ? ok : zero;
            }
        }
    }
    da += kr_xor<16>(da);
    da += kr_xor<32>(da);
    dot = kr_wave_reduce(dot, [](float x, float y) { return x + y; });
    if (q4 == 0) sh.da[mine] = da;
    if (lane == 0) sh.dot[wave] = dot;
    __syncthreads();
    if (wave == 0) {
        double x = sh.da[lane];
        if (lane == 63) x += ((double)sh.dot[0] + sh.dot[1]) + ((double)sh.dot[2] + sh.dot[3]);
        #pragma unroll
        for (int d = 1; d < 64; d *= 2) {
            const double y = __shfl_down(x, d);
            if (lane + d < 64) x += y;
        }
        if (lane < rows) {
            const float gate = lane < n ? g.gate[(row0 + lane) * g.ldg + h] : 0.0f;
            // a constant where the gate is outside its range
            g.dgate[(row0 + lane) * g.H + h] = lane >= n || gate > 0.0f || gate < -10000.0f ? 0.0f : (float)x;
        }
    }
}

// Tokens up to which the chunked form is the recurrent one, too. us, recurrent / chunked, 12
// heads of 64: 8 tokens of 1 stream 12.8 / 12.9, of 64 16 / 20, of 512 88 / 117; 12 tokens 13.4 /
// 13.6, 22 / 20, 123 / 116; 6 heads of 128: 8 tokens 12.4 / 12.7, 24 / 28, 111 / 153.
constexpr int kStepTokens = 8;

// Segments of the time axis, by what a call would take: rounds of workgroups (one a CU
// for D = 128, two for 64) times a segment's chunks, for the sums and for the walk, and
// the join's steps, two or three twelfths of a chunk. A segment has two chunks at least.
// us, one walk / split: 12 heads of 64, 1 x 1024 99 / 38, 1 x 4096 386 / 75, 4 x 1024 100 /
// 59, 8 x 1024 101 / 96; 8 heads of 128 147 / 63, 584 / 122, 151 / 93, 152 / 138.
void split_time(long long heads, int T, int D, bool back, int& seg_chunks, int& segments) {
    const int chunks = (T + kChunk - 1) / kChunk;
    const long long slots = D == 64 ? 512 : 256;
    auto rounds = [&](long long n) { return (n + slots - 1) / slots; };
    const int walks = back ? 2 : 1, step = D == 64 ? 2 : 3;
    seg_chunks = chunks;
    segments = 1;
    long long best = 12 * chunks * rounds(walks * heads);
    for (int n = 2; n <= chunks / 2 && n <= 128 && n * heads <= 2 * slots; n++) {
        const int c = (chunks + n - 1) / n, used = (chunks + c - 1) / c;
        const long long cost = 12ll * c * (rounds((back ? 3 : 2) * heads * used) + rounds(walks * heads * used)) + step * used + 24;
        if (cost < best) {
            best = cost;
            seg_chunks = c;
            segments = used;
        }
    }
}

size_t up256(size_t n) { return (n + 255) / 256 * 256; }

// A call's workspace: for the segments of a time split sums, maps and starts (backward
// sums and ends, too), and for the backward pass states, r, D and w of all chunks.
struct DeltaPlan {
    int seg_chunks, segments;
    size_t sums, maps, starts, back_sums, ends, before, diff, behind, w, total;
};
DeltaPlan delta_plan(int B, int T, int H, int D, bool back) {
    const size_t heads = (size_t)B * H, chunks = (size_t)(T + kChunk - 1) / kChunk;
    const size_t state = heads * D * D * sizeof(float), rows = heads * kChunk * D * sizeof(float);
    DeltaPlan p{};
    split_time((long long)heads, T, D, back, p.seg_chunks, p.segments);
    size_t at = 0;
    auto take = [&](size_t& to, size_t bytes) {
        to = at;
        at += up256(bytes);
    };
    if (p.segments > 1) {
        take(p.sums, p.segments * state);
        take(p.maps, p.segments * state);
        take(p.starts, p.segments * state);
        if (back) take(p.back_sums, p.segments * state);
        if (back) take(p.ends, p.segments * state);
    }
    if (back) {
        take(p.before, (chunks + 1) * state);
        take(p.diff, chunks * rows);
        take(p.behind, chunks * state);
        take(p.w, chunks * rows);
    }
    p.total = at;
    return p;
}

bool shape_ok(int B, int T, int H, int D) {
    return B >= 0 && T >= 0 && H >= 1 && (D == 64 || D == 128) && (long long)B * H <= 1 << 24 && T <= 1 << 30;
}

void place(DeltaArgs& f, BackArgs& g, const DeltaPlan& p, char* ws) {
    auto at = [&](size_t o) { return reinterpret_cast<float*>(ws + o); };
    f.seg_chunks = g.seg_chunks = p.seg_chunks;
    f.segments = g.segments = p.segments;
    f.sums = at(p.sums);
    f.maps = at(p.maps);
    f.starts = at(p.starts);
    g.sums = at(p.back_sums);
    g.ends = at(p.ends);
    f.before = at(p.before);
    f.diff = at(p.diff);
    g.before = f.before;
    g.diff = f.diff;
    g.behind = at(p.behind);
    g.w = at(p.w);
}

template <int D>
int launch_join(const DeltaArgs& f, const BackArgs& g, bool back, hipStream_t s) {
    const int heads = f.B * f.H;
    delta_sums_kernel<D><<<dim3(heads, back ? f.segments : f.segments - 1, back ? 3 : 2), 4 * D, 0, s>>>(f, g);
    KR_LAUNCHED();
    delta_join_kernel<D><<<dim3(heads, D / 16, back ? 2 : 1), 4 * D, 0, s>>>(f, g);
    KR_LAUNCHED();
    return KR_OK;
}

template <int D>
int launch(const DeltaArgs& f, const BackArgs& g, bool chunked, hipStream_t s) {
    const int heads = f.B * f.H;
    if (!chunked) {
        delta_step_kernel<D><<<heads, 4 * D, 0, s>>>(f);
    } else {
        if (f.segments > 1) {
            const int rc = launch_join<D>(f, g, false, s);
            if (rc != KR_OK) return rc;
        }
        delta_chunk_kernel<D><<<dim3(heads, f.segments), 4 * D, 0, s>>>(f);
    }
    KR_LAUNCHED();
    return KR_OK;
}

template <int D>
int launch_back(const DeltaArgs& f, const BackArgs& g, hipStream_t s) {
    const int heads = g.B * g.H, chunks = (g.T + kChunk - 1) / kChunk;
    if (f.segments > 1) {
        const int rc = launch_join<D>(f, g, true, s);
        if (rc != KR_OK) return rc;
    }
    delta_both_kernel<D><<<dim3(heads, f.segments, 2), 4 * D, 0, s>>>(f, g);
    KR_LAUNCHED();
    delta_grad_kernel<D><<<dim3(heads, chunks), 256, 0, s>>>(g);
    KR_LAUNCHED();
    return KR_OK;
}

}  // namespace

extern "C" {

size_t kr_gated_delta_workspace_bytes(int B, int T, int H, int D) {
    if (!shape_ok(B, T, H, D) || B == 0 || T <= kStepTokens) return 0;
    return delta_plan(B, T, H, D, false).total;
}

int kr_gated_delta(int B, int T, int H, int D, const uint16_t* q, long long ldq, const uint16_t* k, long long ldk,
                   const uint16_t* v, long long ldv, const float* log_decay, long long ldg, const float* beta,
                   long long ldb, const int32_t* lens, float* state, uint16_t* y, long long ldy, int chunked, void* ws,
                   size_t ws_bytes, void* stream) {
    KR_REQUIRE(shape_ok(B, T, H, D), "kr_gated_delta: bad shape B=%d T=%d H=%d D=%d (D: 64 or 128)", B, T, H, D);
    const long long C = (long long)H * D;
    KR_REQUIRE(ldq >= C && ldk >= C && ldv >= C && ldy >= C && (ldq | ldk | ldv | ldy) % 8 == 0,
               "kr_gated_delta: token strides must be multiples of 8 and at least H * D = %lld", C);
    KR_REQUIRE(ldg >= H && ldb >= H, "kr_gated_delta: strides of log_decay and beta must be at least H = %d", H);
    if (B == 0 || T == 0) return KR_OK;
    KR_REQUIRE(q && k && v && log_decay && beta && state && y, "kr_gated_delta: null pointer");
    KR_REQUIRE((((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)state | (uintptr_t)y) & 15) == 0,
               "kr_gated_delta: q, k, v, state and y must be 16-byte aligned");
    const bool chunks = chunked && T > kStepTokens;
    const DeltaPlan p = chunks ? delta_plan(B, T, H, D, false) : DeltaPlan{};
    KR_REQUIRE(p.total == 0 || (ws && ws_bytes >= p.total && ((uintptr_t)ws & 15) == 0),
               "kr_gated_delta: workspace of %zu bytes, %zu needed (16-byte aligned)", ws_bytes, p.total);
    DeltaArgs g{};
    g.q = reinterpret_cast<const kr_half*>(q);
    g.k = reinterpret_cast<const kr_half*>(k);
    g.v = reinterpret_cast<const kr_half*>(v);
    g.ldq = ldq;
    g.ldk = ldk;
    g.ldv = ldv;
    g.gate = log_decay;
    g.beta = beta;
    g.ldg = ldg;
    g.ldb = ldb;
    g.lens = lens;
    g.state = state;
    g.y = reinterpret_cast<kr_half*>(y);
    g.ldy = ldy;
    g.B = B;
    g.T = T;
    g.H = H;
    BackArgs none{};
    place(g, none, p, static_cast<char*>(ws));
    return D == 64 ? launch<64>(g, none, chunks, kr_stream(stream)) : launch<128>(g, none, chunks, kr_stream(stream));
}

size_t kr_gated_delta_backward_workspace_bytes(int B, int T, int H, int D) {
    if (!shape_ok(B, T, H, D) || B == 0 || T == 0) return 0;
    return delta_plan(B, T, H, D, true).total;
}

int kr_gated_delta_backward(int B, int T, int H, int D, const uint16_t* q, long long ldq, const uint16_t* k,
                            long long ldk, const uint16_t* v, long long ldv, const float* log_decay, long long ldg,
                            const float* beta, long long ldb, const int32_t* lens, const float* state,
                            const uint16_t* dy, long long ldy, const float* dstate, uint16_t* dq, uint16_t* dk,
                            uint16_t* dv, float* dlog_decay, float* dbeta, float* dstate0, void* ws, size_t ws_bytes,
                            void* stream) {
    KR_REQUIRE(shape_ok(B, T, H, D) && B > 0 && T > 0 && T <= kChunk * 65535,
               "kr_gated_delta_backward: bad shape B=%d T=%d H=%d D=%d (D: 64 or 128, T: 1..4194240)", B, T, H, D);
    const long long C = (long long)H * D;
    KR_REQUIRE(ldq >= C && ldk >= C && ldv >= C && ldy >= C && (ldq | ldk | ldv | ldy) % 8 == 0,
               "kr_gated_delta_backward: token strides must be multiples of 8 and at least H * D = %lld", C);
    KR_REQUIRE(ldg >= H && ldb >= H, "kr_gated_delta_backward: strides of log_decay and beta must be at least H = %d", H);
    KR_REQUIRE(q && k && v && log_decay && beta && state && dy && dq && dk && dv && dlog_decay && dbeta && dstate0,
               "kr_gated_delta_backward: null pointer");
    KR_REQUIRE((((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)state | (uintptr_t)dy | (uintptr_t)dstate |
                 (uintptr_t)dq | (uintptr_t)dk | (uintptr_t)dv | (uintptr_t)dstate0) & 15) == 0,
               "kr_gated_delta_backward: all but log_decay, beta, lens and their gradients must be 16-byte aligned");
    const DeltaPlan p = delta_plan(B, T, H, D, true);
    KR_REQUIRE(ws && ws_bytes >= p.total && ((uintptr_t)ws & 255) == 0,
               "kr_gated_delta_backward: workspace of %zu bytes, %zu needed (256-byte aligned)", ws_bytes, p.total);
    DeltaArgs f{};
    f.q = reinterpret_cast<const kr_half*>(q);
    f.k = reinterpret_cast<const kr_half*>(k);
    f.v = reinterpret_cast<const kr_half*>(v);
    f.ldq = ldq;
    f.ldk = ldk;
    f.ldv = ldv;
    f.gate = log_decay;
    f.beta = beta;
    f.ldg = ldg;
    f.ldb = ldb;
    f.lens = lens;
    f.state = const_cast<float*>(state);          // only read where states are kept
    f.B = B;
    f.T = T;
    f.H = H;
    BackArgs g{};
    g.q = f.q;
    g.k = f.k;
    g.dy = reinterpret_cast<const kr_half*>(dy);
    g.ldq = ldq;
    g.ldk = ldk;
    g.ldy = ldy;
    g.gate = log_decay;
    g.beta = beta;
    g.ldg = ldg;
    g.ldb = ldb;
    g.lens = lens;
    g.dstate = dstate;
    g.dstate0 = dstate0;
    place(f, g, p, static_cast<char*>(ws));
    g.dq = reinterpret_cast<kr_half*>(dq);
    g.dk = reinterpret_cast<kr_half*>(dk);
    g.dv = reinterpret_cast<kr_half*>(dv);
    g.dgate = dlog_decay;
    g.dbeta = dbeta;
    g.B = B;
    g.T = T;
    g.H = H;
    return D == 64 ? launch_back<64>(f, g, kr_stream(stream)) : launch_back<128>(f, g, kr_stream(stream));
}

}  // extern "C"
