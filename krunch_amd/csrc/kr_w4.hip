// Products with 4-bit weights: x [M, K] fp16 times a [K, N] weight held as
// integers q in -8..7 with one fp16 scale per output channel and group of 32,
// 64 or 128 inputs (K % 32 == 0).
//
//   y[m, n] = sum_g s[g, n] * c_g,   c_g = sum_{k in group g} q[n, k] x[m, k]
//
// q x has at most 15 significant bits, so c_g is a chain of exact products on
// v_mfma_f32_16x16x32_f16 (k ascending, from zero), and the scale is applied in
// fp32. Reduction contract, whatever the kernel: y = fma(s_g, c_g, y) over the
// groups in order, from zero; so a row has the same bits for any M.
//
// Layout (kr_w4_bytes): blocks of 16 outputs x 128 inputs, 1 KB, (N / 16) major
// and K / 128 minor. Lane l holds 4 words, word c the inputs 32 c + 8 (l / 16)
// .. + 7 of output l % 16, as the MFMA operand of k-step c: a wave's load of a
// block is one contiguous KB, 16 bytes a lane. Nibbles are q + 8, in the order
// 0, 2, 4, 6, 1, 3, 5, 7 from the low one up: two ANDs (bits 0..3 and 4..7 of
// each half) and one shift give fp16 pairs in operand order, by their place in
// the mantissa of 1024 and of 64 (a published way to make floats of small
// integers), and one packed addition takes 1024 + 8 or 64 + 8 off, exactly: 9
// operations for 8 weights. Padding is q = 0, scale 0.
#include "kr_gemm_epilogue.h"
#include "krunch_hip.h"

namespace {

constexpr int kBlockK = 128;
constexpr int kMaxSplit = 8;                 // waves that share a tile

typedef kr_half kr_half2 __attribute__((ext_vector_type(2)));
typedef kr_half4 kr_half4_any __attribute__((aligned(2)));
typedef kr_float4 kr_float4_any __attribute__((aligned(4)));

struct W4Args {
    const kr_half* x;
    long long ldx;
    const kr_int4* q;
    const kr_half* scales;    // [groups, n16]
    int n16;
    kr_gemm_args o;           // out, ldo, res, gate, M, N, K
};

// The 8 weights of a word as an MFMA operand. The masks and magic numbers are
// held in registers the compiler does not see into: as literals (one per
// instruction) they make AND and OR two operations instead of v_and_or_b32.
struct Unpacker {
    uint32_t low, high, magic_low, magic_high;
    __device__ __forceinline__ Unpacker() {
        __asm__("s_mov_b32 %0, 0x000f000f" : "=s"(low));
        __asm__("s_mov_b32 %0, 0x00f000f0" : "=s"(high));
        __asm__("v_mov_b32 %0, 0x64006400" : "=v"(magic_low));
        __asm__("v_mov_b32 %0, 0x54005400" : "=v"(magic_high));
    }
    __device__ __forceinline__ kr_half8 operator()(uint32_t w) const {
        const kr_half2 k1024 = {(kr_half)-1032.0f, (kr_half)-1032.0f};
        const kr_half2 k64 = {(kr_half)-72.0f, (kr_half)-72.0f};
        const uint32_t v = w >> 8;
        const kr_half2 a = __builtin_bit_cast(kr_half2, (w & low) | magic_low) + k1024;
        const kr_half2 b = __builtin_bit_cast(kr_half2, (w & high) | magic_high) + k64;
        const kr_half2 c = __builtin_bit_cast(kr_half2, (v & low) | magic_low) + k1024;
        const kr_half2 d = __builtin_bit_cast(kr_half2, (v & high) | magic_high) + k64;
        return kr_half8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
    }
};

// Columns n..n+3 of row m; rows of out start at any element.
template <int EP>
__device__ __forceinline__ void store4(const kr_gemm_args& g, int m, int n, kr_float4 acc) {
    if (m >= g.M) return;
    const size_t o = (size_t)m * (size_t)g.ldo + (size_t)n;
    if (n + 3 < g.N && EP == KR_EP_F32) {
        *reinterpret_cast<kr_float4_any*>(reinterpret_cast<float*>(g.out) + o) = acc;
    } else if (n + 3 < g.N && EP == KR_EP_F16) {
        *reinterpret_cast<kr_half4_any*>(reinterpret_cast<kr_half*>(g.out) + o) =
            kr_half4{kr_f16(acc[0]), kr_f16(acc[1]), kr_f16(acc[2]), kr_f16(acc[3])};
    } else {
        #pragma unroll
        for (int r = 0; r < 4; r++)
            if (n + r < g.N) store_one<EP>(g, m, n + r, acc[r]);
    }
}

// Groups [g_begin, g_end) of one 16-output tile against 16 rows, x read from
// memory: each group's chain to take(group, chain). GS = k-steps per group.
template <int GS, typename Take>
__device__ __forceinline__ void tile_groups(const W4Args& g, const Unpacker& unpack, int tile, int g_begin,
                                            int g_end, const kr_half* xr, Take take) {
    constexpr int GPB = 4 / GS;
    const int lane = threadIdx.x & 63;
    const int kb_all = (g.o.K + kBlockK - 1) / kBlockK;
    const kr_int4* q = g.q + ((size_t)tile * kb_all + g_begin / GPB) * 64 + lane;
    for (int g0 = g_begin; g0 < g_end; g0 += GPB, q += 64) {
        const kr_int4 w = *q;
        #pragma unroll
        for (int j = 0; j < GPB; j++) {
            if (g0 + j >= g_end) break;
            kr_float4 c = {0, 0, 0, 0};
            #pragma unroll
            for (int i = 0; i < GS; i++) {
                const int k = (g0 + j) * 32 * GS + 32 * i;
                if (i > 0 && k >= g.o.K) break;
                c = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                    unpack((uint32_t)w[j * GS + i]), *reinterpret_cast<const kr_half8*>(xr + k), c, 0, 0, 0);
            }
            take(g0 + j, c);
        }
    }
}

__device__ __forceinline__ void add_group(kr_half4 s, kr_float4 c, kr_float4& y) {
    #pragma unroll
    for (int r = 0; r < 4; r++) y[r] = __builtin_fmaf((float)s[r], c[r], y[r]);
}

// Up to 16 rows: 16 outputs for a wave, its weights read once, x from the L1.
// With SPLIT, the workgroup's waves share one tile, each a run of its blocks, and
// leave every group's chains (of the rows there are) and scales in LDS, from where
// wave 0 adds them in order, `room` groups at a time; else each wave has a tile of
// its own.
// Bound: latency (a launch, a read of memory, the chains of a wave's blocks).
template <int GS, int EP, bool SPLIT>
__global__ void __launch_bounds__(SPLIT ? 64 * kMaxSplit : 256) w4_rows_kernel(W4Args g, int room) {
    constexpr int GPB = 4 / GS;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
    const int tile = SPLIT ? blockIdx.x : blockIdx.x * waves + wave;
    if (!SPLIT && 16 * tile >= g.n16) return;
    const Unpacker unpack;
    const int m = lane & 15, q4 = lane >> 4, n = 16 * tile + 4 * q4;     // rows past M read the last one
    const kr_half* xr = g.x + (size_t)(m < g.o.M ? m : g.o.M - 1) * g.ldx + 8 * q4;
    const kr_half* sc = g.scales + n;
    auto scales = [&](int i) { return *reinterpret_cast<const kr_half4*>(sc + (size_t)i * g.n16); };
    const int groups = (g.o.K + 32 * GS - 1) / (32 * GS);
    kr_float4 y = {0, 0, 0, 0};
    if constexpr (SPLIT) {
        extern __shared__ kr_float4 chains[];           // [room][4][M], then the scales [room][4]
        const int M = g.o.M;
        kr_half4* held = reinterpret_cast<kr_half4*>(chains + room * 4 * M);
        for (int at = 0; at < groups; at += room) {
            const int end = groups - at < room ? groups : at + room;
            const int run = ((end - at + GPB - 1) / GPB + waves - 1) / waves * GPB;
            const int g0 = at + wave * run, g1 = g0 + run < end ? g0 + run : end;
            tile_groups<GS>(g, unpack, tile, g0, g1, xr, [&](int i, kr_float4 c) {
                const int k = (i - at) * 4 + q4;
                if (m == 0) held[k] = scales(i);
                if (m < M) chains[k * M + m] = c;
            });
            __syncthreads();
            if (wave == 0 && m < M) {
                #pragma unroll 8
                for (int i = 0; i < end - at; i++) add_group(held[i * 4 + q4], chains[(i * 4 + q4) * M + m], y);
            }
            if (end < groups) __syncthreads();
        }
        if (wave == 0) store4<EP>(g.o, m, n, y);
    } else {
        tile_groups<GS>(g, unpack, tile, 0, groups, xr, [&](int i, kr_float4 c) { add_group(scales(i), c, y); });
        store4<EP>(g.o, m, n, y);
    }
}

template <int GS, int EP>
int launch_rows(const W4Args& g, hipStream_t s) {
    const int tiles = g.n16 / 16, blocks = (g.o.K + kBlockK - 1) / kBlockK;
    // 1024 tiles are a wave for each SIMD without a split
    if (blocks > 1 && tiles < 1024) {
        const int waves = blocks < kMaxSplit ? blocks : kMaxSplit;
        const int a_group = 64 * g.o.M + 32;                       // bytes of LDS
        const int most = 65536 / (a_group * (4 / GS));             // blocks at a time
        const int turns = (blocks + most - 1) / most;
        const int room = (blocks + turns - 1) / turns * (4 / GS);
        w4_rows_kernel<GS, EP, true><<<tiles, 64 * waves, (size_t)room * a_group, s>>>(g, room);
    } else {
        w4_rows_kernel<GS, EP, false><<<(tiles + 3) / 4, 256, 0, s>>>(g, 0);
    }
    KR_LAUNCHED();
    return KR_OK;
}

// More rows, any K: a workgroup has 64 outputs, 16 for each of its 4 waves, against
// 32 rows. x goes through LDS in blocks of 128 inputs (two buffers, one barrier a
// block); the weights go straight to their wave's registers, and are unpacked
// once for the 32 rows. Both are asked for kTileAhead blocks ahead.
// Bound: latency, where the kernels below have too few units of work.
// us by blocks ahead, 1 / 3: 64 x 768 x 768, groups of 32 6.2 / 5.5, 64 5.4 / 4.8,
// 128 5.8 / 5.7; 64 x 2048 x 8192 14.0 / 11.6, 11.9 / 10.0, 13.1 / 14.8. Tiles of
// 64 x 64 and 128 x 64 are slower on both (8.0 / 7.5 and 11.1 at groups of 32).
template <int GS, int EP>
__global__ void __launch_bounds__(256, 2) w4_tile_kernel(W4Args g) {
    constexpr int MT = 2, ROWS = 16 * MT;
    constexpr int kTileAhead = GS == 4 ? 1 : 3;
    constexpr int GPB = 4 / GS;                             // groups per block
    __shared__ kr_half8 xs[2][ROWS * 16];                   // unit c of row m at 16 m + (c ^ m % 16)
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int l16 = lane & 15, q4 = lane >> 4;
    const int tiles = g.n16 / 16, tile = blockIdx.x * 4 + wave;
    const int t_read = tile < tiles ? tile : tiles - 1;               // past N: the last tile, not stored
    const int m0 = blockIdx.y * ROWS;
    const int kb_all = (g.o.K + kBlockK - 1) / kBlockK, groups = (g.o.K + 32 * GS - 1) / (32 * GS);
    const Unpacker unpack;
    const kr_int4* qp = g.q + (size_t)t_read * kb_all * 64 + lane;
    const kr_half* sp = g.scales + 16 * t_read + 4 * q4;
    const kr_half* xp[MT];
    #pragma unroll
    for (int i = 0; i < MT; i++) {
        const int m = m0 + 16 * i + tid / 16;                         // past M: the last row, not stored
        xp[i] = g.x + (size_t)(m < g.o.M ? m : g.o.M - 1) * g.ldx;
    }
    kr_half8 xv[kTileAhead][MT];
    kr_int4 w[kTileAhead];
    kr_half4 sc[kTileAhead][GPB];
    auto fetch = [&](int kb, kr_half8 (&xn)[MT], kr_int4& wn, kr_half4 (&sn)[GPB]) {
        if (kb >= kb_all) return;
        // inputs past K are zeros, and so the products with them, whatever scale is read
        const int k = kb * kBlockK + 8 * (tid & 15);
        #pragma unroll
        for (int i = 0; i < MT; i++) {
            xn[i] = kr_half8{0, 0, 0, 0, 0, 0, 0, 0};
            if (k < g.o.K) xn[i] = *reinterpret_cast<const kr_half8*>(xp[i] + k);
        }
        wn = qp[(size_t)kb * 64];
        #pragma unroll
        for (int j = 0; j < GPB; j++) {
            const int gi = kb * GPB + j < groups ? kb * GPB + j : groups - 1;
            sn[j] = *reinterpret_cast<const kr_half4*>(sp + (size_t)gi * g.n16);
        }
    };
    kr_float4 y[MT];
    #pragma unroll
    for (int t = 0; t < MT; t++) y[t] = kr_float4{0, 0, 0, 0};
    #pragma unroll
    for (int a = 0; a < kTileAhead; a++) fetch(a, xv[a], w[a], sc[a]);
    for (int kb = 0; kb < kb_all; kb++) {
        kr_half8* xb = xs[kb & 1];
        #pragma unroll
        for (int i = 0; i < MT; i++) xb[(16 * i + tid / 16) * 16 + ((tid & 15) ^ (tid / 16))] = xv[0][i];
        const kr_int4 wc = w[0];
        kr_half4 sg[GPB];
        #pragma unroll
        for (int j = 0; j < GPB; j++) sg[j] = sc[0][j];
        #pragma unroll
        for (int a = 1; a < kTileAhead; a++) {
            #pragma unroll
            for (int i = 0; i < MT; i++) xv[a - 1][i] = xv[a][i];
            w[a - 1] = w[a];
            #pragma unroll
            for (int j = 0; j < GPB; j++) sc[a - 1][j] = sc[a][j];
        }
        fetch(kb + kTileAhead, xv[kTileAhead - 1], w[kTileAhead - 1], sc[kTileAhead - 1]);
        __syncthreads();      // and with it, every wave is done with the buffer of kb - 1
        kr_float4 c[MT];
        #pragma unroll
        for (int s = 0; s < 4; s++) {
            const kr_half8 a = unpack((uint32_t)wc[s]);
            #pragma unroll
            for (int t = 0; t < MT; t++) {
                if (s % GS == 0) c[t] = kr_float4{0, 0, 0, 0};
                c[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                    a, xb[(16 * t + l16) * 16 + ((4 * s + q4) ^ l16)], c[t], 0, 0, 0);
            }
            if ((s + 1) % GS == 0) {
                #pragma unroll
                for (int r = 0; r < 4; r++) {
                    const float f = (float)sg[s / GS][r];
                    #pragma unroll
                    for (int t = 0; t < MT; t++) y[t][r] = __builtin_fmaf(f, c[t][r], y[t][r]);
                }
            }
        }
    }
    if (tile < tiles) {
        #pragma unroll
        for (int t = 0; t < MT; t++) store4<EP>(g.o, m0 + 16 * t + l16, 16 * tile + 4 * q4, y[t]);
    }
}

template <int GS, int EP>
int launch_tile(const W4Args& g, hipStream_t s) {
    // outputs in steps of 8 workgroups: those of an XCD (every eighth) keep
    // their weights in its L2 from one row tile to the next
    const int groups = (g.n16 / 16 + 3) / 4;
    const int gx = groups >= 8 ? (groups + 7) / 8 * 8 : groups;
    w4_tile_kernel<GS, EP><<<dim3(gx, (g.o.M + 31) / 32), 256, 0, s>>>(g);
    KR_LAUNCHED();
    return KR_OK;
}

// Rows held: a workgroup has all of K of 16 MT rows in LDS, zeros past K, and its
// waves take units of 16 NT outputs one after another, each on its own: no barrier
// after the rows are in. Weights come kAhead blocks ahead into registers.
// Bound with 64 rows: the VALU's 3.6 operations a product (2 to unpack, shared by four
// row tiles, 1 to scale) beside a matrix unit at 30%, the waits of three waves a SIMD
// (43% of their time) and the last units of a range, which leave waves idle. Measured on
// MI355X, 512 x 768 x 50277 at groups of 32 / 64 / 128: 76 / 62 / 49 us (0.81 PF/s at 128; the
// rows of x held by 8 waves 53, through LDS a tile at a time 76), 2000 rows 250 / 204 /
// 192. Rows of 50277 fp16 start anywhere in a line: 50272 takes 45 us. Stores without
// bounds, with a quarter of the operations, change nothing (50).
// Bound with 16 rows: latency, about 4.5 us beside what the weights take.
constexpr int kHeldUnits = 163840 / 16;      // all of a CU's LDS: one workgroup each

template <int NT, int MT, int GS, int EP, int kAhead, int kHeldWaves>
__global__ void __launch_bounds__(64 * kHeldWaves, kHeldWaves / 4) w4_held_kernel(W4Args g, int ranges) {
    constexpr int GPB = 4 / GS;
    __shared__ kr_half8 xs[kHeldUnits];      // unit c of row m of block b at 16 (16 MT b + m) + (c ^ m % 16)
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int l16 = lane & 15, q4 = lane >> 4;
    // with ranges of outputs in eights, the workgroups of one are 8 apart: on one XCD,
    // whose L2 then has the weights for all of them
    const int row_tiles = (g.o.M + 16 * MT - 1) / (16 * MT);
    const int range = ranges % 8 ? blockIdx.x % ranges : blockIdx.x % 8 + blockIdx.x / 8 / row_tiles * 8;
    const int m0 = (ranges % 8 ? blockIdx.x / ranges : blockIdx.x / 8 % row_tiles) * 16 * MT;
    const int kb_all = (g.o.K + kBlockK - 1) / kBlockK, groups = (g.o.K + 32 * GS - 1) / (32 * GS);
    const int tiles = g.n16 / 16, units = (tiles + NT - 1) / NT;
    for (int i = tid; i < 16 * MT * kb_all * 16; i += 64 * kHeldWaves) {
        const int m = i / (kb_all * 16), c = i - m * (kb_all * 16);   // neighbours along a row
        kr_half8 v = {0, 0, 0, 0, 0, 0, 0, 0};
        if (m0 + m < g.o.M && 8 * c < g.o.K)
            v = *reinterpret_cast<const kr_half8*>(g.x + (size_t)(m0 + m) * g.ldx + 8 * c);
        xs[16 * (c / 16 * 16 * MT + m) + ((c ^ m) & 15)] = v;
    }
    __syncthreads();
    const Unpacker unpack;
    const kr_half8* xl[4];
    #pragma unroll
    for (int s = 0; s < 4; s++) xl[s] = xs + l16 * 16 + ((4 * s + q4) ^ l16);
    const int step = ranges * kHeldWaves;
    int unit = range + ranges * wave;
    if (unit >= units) return;

    // blocks in flight: next_unit, next_kb is the first not yet asked for
    kr_int4 w[kAhead][NT];
    kr_half4 sc[kAhead][NT][GPB];
    int next_unit = unit, next_kb = 0;
    const kr_int4* qp[NT];
    const kr_half* sp[NT];
    auto point = [&]() {
        #pragma unroll
        for (int i = 0; i < NT; i++) {
            const int tile = next_unit * NT + i < tiles ? next_unit * NT + i : tiles - 1;
            qp[i] = g.q + (size_t)tile * kb_all * 64 + lane;
            sp[i] = g.scales + 16 * tile + 4 * q4;
        }
    };
    auto fetch = [&](kr_int4 (&wn)[NT], kr_half4 (&sn)[NT][GPB]) {
        if (next_unit >= units) return;
        #pragma unroll
        for (int i = 0; i < NT; i++) {
            wn[i] = qp[i][next_kb * 64];
            #pragma unroll
            for (int j = 0; j < GPB; j++) {
                const int gi = next_kb * GPB + j < groups ? next_kb * GPB + j : groups - 1;   // the products are 0
                sn[i][j] = *reinterpret_cast<const kr_half4*>(sp[i] + (size_t)gi * g.n16);
            }
        }
        if (++next_kb == kb_all) {
            next_kb = 0;
            next_unit += step;
            point();
        }
    };
    point();
    #pragma unroll
    for (int a = 0; a < kAhead; a++) fetch(w[a], sc[a]);
    for (; unit < units; unit += step) {
        kr_float4 y[NT][MT];
        #pragma unroll
        for (int i = 0; i < NT; i++)
            #pragma unroll
            for (int t = 0; t < MT; t++) y[i][t] = kr_float4{0, 0, 0, 0};
        for (int kb = 0; kb < kb_all; kb++) {
            kr_int4 wc[NT];
            kr_half4 sg[NT][GPB];
            #pragma unroll
            for (int i = 0; i < NT; i++) {
                wc[i] = w[0][i];
                #pragma unroll
                for (int j = 0; j < GPB; j++) sg[i][j] = sc[0][i][j];
                #pragma unroll
                for (int a = 1; a < kAhead; a++) {
                    w[a - 1][i] = w[a][i];
                    #pragma unroll
                    for (int j = 0; j < GPB; j++) sc[a - 1][i][j] = sc[a][i][j];
                }
            }
            fetch(w[kAhead - 1], sc[kAhead - 1]);
            kr_float4 c[NT][MT];
            #pragma unroll
            for (int s = 0; s < 4; s++) {
                kr_half8 x[MT];
                #pragma unroll
                for (int t = 0; t < MT; t++) x[t] = xl[s][256 * (MT * kb + t)];
                #pragma unroll
                for (int i = 0; i < NT; i++) {
                    const kr_half8 a = unpack((uint32_t)wc[i][s]);
                    #pragma unroll
                    for (int t = 0; t < MT; t++) {
                        if (s % GS == 0) c[i][t] = kr_float4{0, 0, 0, 0};
                        c[i][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, x[t], c[i][t], 0, 0, 0);
                    }
                }
                if ((s + 1) % GS == 0) {
                    #pragma unroll
                    for (int i = 0; i < NT; i++)
                        #pragma unroll
                        for (int r = 0; r < 4; r++) {
                            const float f = (float)sg[i][s / GS][r];
                            #pragma unroll
                            for (int t = 0; t < MT; t++) y[i][t][r] = __builtin_fmaf(f, c[i][t][r], y[i][t][r]);
                        }
                    // or the next group's x comes early and registers spill (2000 rows 220 us)
                    if (GS == 2) __builtin_amdgcn_sched_barrier(0);
                }
            }
        }
        #pragma unroll
        for (int t = 0; t < MT; t++)
            #pragma unroll
            for (int i = 0; i < NT; i++)
                if (unit * NT + i < tiles)
                    store4<EP>(g.o, m0 + 16 * t + l16, 16 * (unit * NT + i) + 4 * q4, y[i][t]);
    }
}

// Whether 16 MT rows of this K fit, and give every wave of 256 workgroups a unit.
bool held_fits(const W4Args& g, int MT) {
    return (long long)(g.o.K + kBlockK - 1) / kBlockK * 16 * 16 * MT <= kHeldUnits;
}
bool held_fills(const W4Args& g, int NT, int MT, int waves) {
    return held_fits(g, MT) && (long long)((g.n16 / 16 + NT - 1) / NT) * ((g.o.M + 16 * MT - 1) / (16 * MT)) >=
                                   256 * waves;
}

template <int NT, int MT, int GS, int EP, int kAhead, int kHeldWaves>
int launch_held(const W4Args& g, hipStream_t s) {
    const int row_tiles = (g.o.M + 16 * MT - 1) / (16 * MT);
    const int units = (g.n16 / 16 + NT - 1) / NT;
    // one workgroup a CU; in eights where that leaves out few of them
    int ranges = row_tiles < 256 ? 256 / row_tiles : 1;
    const int most = (units + kHeldWaves - 1) / kHeldWaves;
    if (ranges > most) ranges = most;
    if (16 * (ranges / 8 * 8) >= 15 * ranges) ranges = ranges / 8 * 8;
    w4_held_kernel<NT, MT, GS, EP, kAhead, kHeldWaves><<<ranges * row_tiles, 64 * kHeldWaves, 0, s>>>(g, ranges);
    KR_LAUNCHED();
    return KR_OK;
}

// Kernel by the work there is, us on MI355X at groups of 32 / 64 / 128:
//   up to 16 rows, fewer than 1536 tiles of 16 outputs: rows, else held (16 x 16).
//     1 x 768 x 16384 rows 5.2 / 5.5 / 4.7, held 8.5 / 7.0 / 6.4; 1 x 768 x 32768
//     9.6 / 10.3 / 8.6 and 8.8 / 7.4 / 6.8; 16 x 768 x 50277 17.1 / 17.1 / 15.9 and
//     11.1 / 9.7 / 9.2.
//   more rows: held with 64 rows, else with 32, where that gives each of the 12
//     waves of 256 workgroups a unit of 32 outputs; else tiles. 512 x 768 x 16384
//     (4096 units of 64 rows) held 64 26.3 / 20.4 / 18.2, held 32 29.1 / 22.5 / 20.2,
//     tiles 34.7 / 29.5 / 25.7; 512 x 768 x 8192 (2048 units of 64 rows, 4096 of 32) held
//     64 19.4 / 16.4 / 15.0, held 32 15.5 / 12.6 / 12.0, tiles 18.7 / 16.4 / 14.7; 128 x
//     768 x 16384 (2048 of 32) held 32 13.1 / 11.4 / 10.7, tiles 11.4 / 10.0 / 9.2.
template <int GS, int EP>
int launch_by_rows(const W4Args& g, hipStream_t s) {
    if (g.o.M <= 16) {
        if (g.n16 / 16 >= 1536 && held_fits(g, 1)) return launch_held<1, 1, GS, EP, 3, 16>(g, s);
        return launch_rows<GS, EP>(g, s);
    }
    if (held_fills(g, 2, 4, 12)) return launch_held<2, 4, GS, EP, 1, 12>(g, s);
    if (held_fills(g, 2, 2, 12)) return launch_held<2, 2, GS, EP, 1, 12>(g, s);
    return launch_tile<GS, EP>(g, s);
}

template <int EP>
int launch_by_group(const W4Args& g, int group, hipStream_t s) {
    if (group == 32) return launch_by_rows<1, EP>(g, s);
    if (group == 64) return launch_by_rows<2, EP>(g, s);
    return launch_by_rows<4, EP>(g, s);
}

// One thread per output and group. s = fp16(amax / 7); q = x / s to the nearest
// integer, ties to even, at most 7 in size; 0 where s is 0 (a group of zeros, or
// of values under 7 * 2^-25). The quotient of two fp16 values lies on a tie or
// at least 2^-12 of itself from one, so dividing in fp32 first changes no q. A
// group with an infinity or NaN gets a NaN scale. W is read at
// W[k * ldk + n * ldn]; one of the two is 1 in use. Bound: memory with ldn = 1 (768 x
// 50277 83 us), requests with ldk = 1, where a wave's reads lie in 64 rows (1.05 ms).
__global__ void __launch_bounds__(256) w4_quantize_kernel(const kr_half* __restrict__ W, long long ldk,
                                                          long long ldn, int N, int K, int group,
                                                          uint32_t* __restrict__ q,
                                                          kr_half* __restrict__ scales, int n16) {
    const int n = blockIdx.x * 256 + threadIdx.x;
    if (n >= n16) return;
    const int kb_all = (K + kBlockK - 1) / kBlockK;
    const int k0 = blockIdx.y * group;
    const int count = n < N ? (K - k0 < group ? K - k0 : group) : 0;
    const kr_half* w = W + (size_t)(n < N ? n : 0) * (size_t)ldn + (size_t)k0 * (size_t)ldk;
    float amax = 0.0f;
    bool finite = true;
    for (int i = 0; i < count; i++) {
        const float a = fabsf((float)w[(size_t)i * (size_t)ldk]);
        finite = finite && a <= 65504.0f;
        amax = fmaxf(amax, a);
    }
    const kr_half sh = finite ? kr_f16(amax / 7.0f) : (kr_half)NAN;
    const float s = (float)sh;
    if (k0 < K) scales[(size_t)blockIdx.y * n16 + n] = sh;
    for (int i = 0; i < group; i += 8) {
        const int k = k0 + i;
        uint32_t word = 0;
        #pragma unroll
        for (int e = 0; e < 8; e++) {
            float v = 0.0f;
            if (i + e < count && s > 0.0f)
                v = fminf(fmaxf(__builtin_rintf((float)w[(size_t)(i + e) * (size_t)ldk] / s), -7.0f), 7.0f);
            word |= (uint32_t)((int)v + 8) << (4 * (e / 2 + 4 * (e % 2)));
        }
        const size_t block = (size_t)(n >> 4) * kb_all + k / kBlockK;
        q[(block * 64 + (n & 15) + 16 * (k % 32 / 8)) * 4 + k % kBlockK / 32] = word;
    }
}

int check_w4(const char* who, int N, int K, int group) {
    KR_REQUIRE(N >= 1 && N <= (1 << 30), "%s: N=%d", who, N);
    KR_REQUIRE(K >= 32 && K % 32 == 0 && K <= (1 << 20), "%s: K=%d must be a multiple of 32 up to %d", who, K,
               1 << 20);
    KR_REQUIRE(group == 32 || group == 64 || group == 128, "%s: group=%d must be 32, 64 or 128", who,
               group);
    return KR_OK;
}

}  // namespace

extern "C" {

size_t kr_w4_bytes(int N, int K) {
    if (N < 1 || K < 32 || K % 32) return 0;
    return ((size_t)N + 15) / 16 * (((size_t)K + kBlockK - 1) / kBlockK) * 1024;
}

int kr_quantize_w4(const uint16_t* W, long long ldk, long long ldn, int N, int K, int group, void* q,
                   uint16_t* scales, void* stream) {
    if (const int rc = check_w4("kr_quantize_w4", N, K, group)) return rc;
    KR_REQUIRE(W && q && scales, "kr_quantize_w4: null pointer");
    KR_REQUIRE(((uintptr_t)q & 15) == 0 && ((uintptr_t)scales & 7) == 0 && ((uintptr_t)W & 1) == 0,
               "kr_quantize_w4: misaligned pointer");
    KR_REQUIRE(ldk >= 1 && ldn >= 1, "kr_quantize_w4: strides %lld, %lld", ldk, ldn);
    const int n16 = (N + 15) / 16 * 16;
    // every group of the padded K: the last block's padding is written too
    const int groups = (K + kBlockK - 1) / kBlockK * (kBlockK / group);
    w4_quantize_kernel<<<dim3((n16 + 255) / 256, groups), 256, 0, kr_stream(stream)>>>(
        reinterpret_cast<const kr_half*>(W), ldk, ldn, N, K, group, reinterpret_cast<uint32_t*>(q),
        reinterpret_cast<kr_half*>(scales), n16);
    KR_LAUNCHED();
    return KR_OK;
}

int kr_det_matmul_w4(const uint16_t* x, long long ldx, int M, int K, const void* q,
                     const uint16_t* scales, int group, int N, void* out, long long ldo, int epilogue,
                     const uint16_t* res, const uint16_t* gate, void* stream) {
    if (const int rc = check_w4("kr_det_matmul_w4", N, K, group)) return rc;
    KR_REQUIRE(M >= 0 && M <= (1 << 19), "kr_det_matmul_w4: M=%d must be in 0..%d", M, 1 << 19);
    KR_REQUIRE(ldx >= K && ldx % 8 == 0 && ldo >= N,
               "kr_det_matmul_w4: ldx=%lld must be a multiple of 8 >= K=%d, ldo=%lld >= N=%d", ldx, K,
               ldo, N);
    KR_REQUIRE(epilogue >= KR_EP_F32 && epilogue <= KR_EP_GATED, "kr_det_matmul_w4: epilogue %d",
               epilogue);
    if (M == 0) return KR_OK;
    KR_REQUIRE(x && q && scales && out, "kr_det_matmul_w4: null pointer");
    KR_REQUIRE(epilogue < KR_EP_RESID || res, "kr_det_matmul_w4: epilogue %d needs res", epilogue);
    KR_REQUIRE(epilogue != KR_EP_GATED || gate, "kr_det_matmul_w4: epilogue %d needs gate", epilogue);
    KR_REQUIRE((((uintptr_t)x | (uintptr_t)q) & 15) == 0 && ((uintptr_t)scales & 7) == 0,
               "kr_det_matmul_w4: misaligned pointer (x, q: 16 bytes; scales: 8)");
    W4Args g{};
    g.x = reinterpret_cast<const kr_half*>(x);
    g.ldx = ldx;
    g.q = reinterpret_cast<const kr_int4*>(q);
    g.scales = reinterpret_cast<const kr_half*>(scales);
    g.n16 = (N + 15) / 16 * 16;
    g.o.out = out;
    g.o.ldo = ldo;
    g.o.res = reinterpret_cast<const kr_half*>(res);
    g.o.gate = reinterpret_cast<const kr_half*>(gate);
    g.o.M = M;
    g.o.N = N;
    g.o.K = K;
    const hipStream_t s = kr_stream(stream);
    switch (epilogue) {
        case KR_EP_F32: return launch_by_group<KR_EP_F32>(g, group, s);
        case KR_EP_F16: return launch_by_group<KR_EP_F16>(g, group, s);
        case KR_EP_SIGMOID: return launch_by_group<KR_EP_SIGMOID>(g, group, s);
        case KR_EP_RELUSQ: return launch_by_group<KR_EP_RELUSQ>(g, group, s);
        case KR_EP_RESID: return launch_by_group<KR_EP_RESID>(g, group, s);
        default: return launch_by_group<KR_EP_GATED>(g, group, s);
    }
}

}  // extern "C"
