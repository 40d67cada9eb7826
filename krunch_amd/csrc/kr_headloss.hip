// Softmax cross entropy of a head [V, C] over a large vocabulary, and its
// gradients, without [N, V] logits in memory.
//
//   z = x W';  lse_n = ln sum_v e^(z_nv);  loss_n = lse_n - z_n,target
//   dz_nv = dloss_n (e^(z_nv - lse_n) - [v is n's target]);  dx = dz W;  dW = dz' x
//
// Forward: tiles of z stay in registers and leave as a maximum and a sum per row
// and 64 or 128 columns, which a second kernel joins. Backward: a piece of the
// vocabulary at a time, z again, dz of the piece as fp16 in the workspace, and both
// products that read it in one launch. The floor is three products of 2 N C V (one
// forward); z a second time is what not keeping it costs.
//
// dz enters the matrix units as fp16 (11 bits, as x and W have): it is kept times a
// power of two that brings the largest |dloss| to 2^14..2^15, so that
// probabilities down to 2^-28 of that keep all their bits; what is left of a target's is
// added back, and an fp16 output's own rounding is nearly all of its error. For fp32
// outputs dz is kept in two such parts, 22 bits (7e-7 of dx and dW in 2-norm; with one part
// 3e-5 and 6e-5), and the products have twice the steps: 8192 x 768 x 50277 3,665 us,
// fp16 2,070. Sums are fp32.
#include <algorithm>

#include "kr_common.h"
#include "kr_copy.h"
#include "kr_wave.h"
#include "krunch_hip.h"

namespace {

constexpr float kLog2e = 0x1.715476p+0f, kLn2 = 0x1.62e430p-1f;
typedef short short4v __attribute__((__vector_size__(8)));
typedef __attribute__((address_space(3))) short4v lds_short4;

struct LossArgs {
    const kr_half* x;
    const kr_half* W;                 // [V, C], at the piece's first row
    long long ldx, ldw;
    const int32_t* targets;
    const float* lse;                 // GRAD
    const float* dloss;
    const float* scale;               // [2] up, down
    float2* part;                     // LOSS: [parts][N] maximum, sum
    float* hit;                       // LOSS: [N] the target's z
    kr_half* G;                       // GRAD: [rows][ldg] dz of the piece
    kr_half* G_low;                   // GRAD: what fp16 leaves of them (null: not kept)
    long long ldg;
    float* left;                      // GRAD: [N] what fp16 leaves of the target's dz
    int N, C, V;                      // V: the piece's columns
    int v0, v_all;                    // the piece's first column, the vocabulary
    int rows;                         // GRAD: N rounded up to 64, the rows of G
};

__device__ __forceinline__ void copy16(const void* base, unsigned off, unsigned lds) {
    kr_copy16(base, off, (unsigned)__builtin_amdgcn_readfirstlane((int)lds));
}
// A pointer that all lanes share, as such to the compiler.
template <typename T>
__device__ __forceinline__ const T* shared_by_lanes(const T* p) {
    const uint64_t v = (uint64_t)p;
    return reinterpret_cast<const T*>((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)v) |
                                      (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(v >> 32)) << 32);
}
__device__ __forceinline__ unsigned lds_address(const void* p) {
    return (unsigned)(uintptr_t)(__attribute__((address_space(3))) const char*)p;
}

// LDS place, in 16-byte units, of unit kc (8 k) of row r of an operand whose rows
// lie along k: a copy instruction moves 8 whole 128-byte lines, and 8 rows' units of
// one kc lie on different banks.
__device__ __forceinline__ int row_unit(int r, int kc) { return 8 * r + (kc ^ ((r >> 1) & 7)); }

// The same for W of a tile, 16 of whose rows are read as 8 a + b, a and b 0..3 (or 4 more).
__device__ __forceinline__ int w_swap(int r) { return ((r >> 1) & 1) | ((r >> 2) & 6); }
__device__ __forceinline__ int w_unit(int r, int kc) { return 8 * r + (kc ^ w_swap(r)); }

// Tile of the launch's virtual workgroup vb: an eighth of a grouped order for each XCD.
__device__ __forceinline__ bool tile_of(int gy, int gx, int vb, int group_m, int& m_t, int& n_t) {
    const int T = gx * gy, per = (T + 7) / 8;
    const int t = (vb & 7) * per + (vb >> 3);
    if (t >= T || (vb >> 3) >= per) return false;
    const int in_group = group_m * gx;
    const int first_m = (t / in_group) * group_m;
    const int gm = min(gy - first_m, group_m);
    const int r = t % in_group;
    m_t = first_m + r % gm;
    n_t = r / gm;
    return true;
}

// ---------------------------------------------------------------------------
// z = x W' in tiles of (64 WM) x (16 TN WN), a wave for each 64 x 16 TN. Steps of 64 k
// through two LDS stages, copied asynchronously one step ahead, into the next tile. The
// matrix unit gets W' x', so a lane has 4 columns of a row; W's rows go in in an
// order that makes them 8 consecutive columns over two of its tiles.
// Bound, at 256 x 256: the copies, one step ahead (a step takes 4,400 cycles, its matrix
// instructions 2,050, LDS reads 770), and the epilogue that nothing overlaps (an
// exponential each). Measured on MI355X, 8192 x 768 x 50277: losses 580 us
// (1.09 PF/s; a library's product of the same sizes 703, 8192^3 at 1.16), dz 156 us for
// 10240 columns (0.83 PF/s, 168 MB stored). A bank conflict in every read of W cost 40 us of
// the losses, a cursor over tiles that allows more stages 25. At 128 x 128, two workgroups
// a CU: 30001 x 512 x 256 15.5 us, of which 6 are its 31 MB (64 x 256 tiles 16, 64 x 128
// 23, 128 x 64 25).
// ---------------------------------------------------------------------------
template <int N>
__device__ __forceinline__ void wait_copies() { asm volatile("s_waitcnt vmcnt(%0)" :: "n"(N) : "memory"); }

template <int WM, int WN, int TN, bool GRAD>
__global__ void __launch_bounds__(64 * WM * WN, WM * WN >= 8 ? 1 : 2) logits_kernel(LossArgs g, int n_virtual,
                                                                                 int group_m) {
    constexpr int BM = 64 * WM, BN = 16 * TN * WN, WAVES = WM * WN;
    constexpr int COPIES = (BM + BN) / 8 / WAVES;
    static_assert((BM + BN) / 8 % WAVES == 0 && TN % 4 == 0, "tile");
    constexpr int STAGE = (BM + BN) * 8;                  // 16-byte units
    __shared__ __attribute__((aligned(1024))) kr_half8 ring[2 * STAGE];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave / WN, wn = wave % WN;
    const int lr = lane & 15, lq = lane >> 4;
    const int gy = ((GRAD ? g.rows : g.N) + BM - 1) / BM, gx = (g.V + BN - 1) / BN;
    const int KS = g.C / 64;
    const unsigned ring_base = lds_address(ring);
    auto issue = [&](int m_t, int n_t, int ks, int q) {
        const kr_half* xa = g.x + (long long)m_t * BM * g.ldx;
        const kr_half* wa = g.W + (long long)n_t * BN * g.ldw;
        const unsigned so = ring_base + (unsigned)((q & 1) * STAGE * 16);
        #pragma unroll
        for (int i = 0; i < COPIES; i++) {
            const int j = wave * COPIES + i;              // 8 rows of the stage
            const bool a = j < BM / 8;
            const int row = 8 * (a ? j : j - BM / 8) + (lane >> 3);
            const int last = a ? g.N - 1 - m_t * BM : g.V - 1 - n_t * BN;
            const int kc = (lane & 7) ^ (a ? (row >> 1) & 7 : w_swap(row));
            const unsigned off = (unsigned)max(min(row, last), 0) * (unsigned)(2 * (a ? g.ldx : g.ldw)) +
                                 (unsigned)(16 * kc + 128 * ks);
            copy16(a ? xa : wa, off, so + 1024u * (unsigned)j);
        }
    };
    int vb = blockIdx.x, m_t, n_t;
    if (!tile_of(gy, gx, vb, group_m, m_t, n_t)) return;
    int q = 0;
    issue(m_t, n_t, 0, 0);
    while (true) {
        int nm_t = 0, nn_t = 0;
        const bool has_next =
            vb + (int)gridDim.x < n_virtual && tile_of(gy, gx, vb + (int)gridDim.x, group_m, nm_t, nn_t);
        kr_float4 acc[4][TN];
        #pragma unroll
        for (int i = 0; i < 4; i++)
            #pragma unroll
            for (int t = 0; t < TN; t++) acc[i][t] = kr_float4{0, 0, 0, 0};
        #pragma unroll 1
        for (int ks = 0; ks < KS; ks++, q++) {
            wait_copies<0>();
            __syncthreads();   // every wave's copies are in; the step before is read
            if (ks + 1 < KS) issue(m_t, n_t, ks + 1, q + 1);
            else if (has_next) issue(nm_t, nn_t, 0, q + 1);
            const kr_half8* As = ring + (q & 1) * STAGE;
            const kr_half8* Ws = As + BM * 8;
            #pragma unroll
            for (int kb = 0; kb < 2; kb++) {
                kr_half8 a[4];
                #pragma unroll
                for (int i = 0; i < 4; i++) a[i] = As[row_unit(64 * wm + 16 * i + lr, 4 * kb + lq)];
                #pragma unroll
                for (int th = 0; th < TN / 4; th++) {
                    __builtin_amdgcn_sched_barrier(0);    // four W fragments at a time (registers)
                    kr_half8 w[4];
                    #pragma unroll
                    for (int t = 0; t < 4; t++) {
                        const int row = 16 * TN * wn + 32 * (2 * th + t / 2) + 8 * (lr >> 2) + 4 * (t & 1) + (lr & 3);
                        w[t] = Ws[w_unit(row, 4 * kb + lq)];
                    }
                    __builtin_amdgcn_sched_barrier(0);
                    #pragma unroll
                    for (int i = 0; i < 4; i++)
                        #pragma unroll
                        for (int t = 0; t < 4; t++)
                            acc[i][4 * th + t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                                w[t], a[i], acc[i][4 * th + t], 0, 0, 0);
                }
            }
        }
        // lane: row 64 wm + 16 i + lr; acc[i][t][r] column 16 TN wn + 32 (t / 2) + 8 lq + 4 (t % 2) + r
        const int first = n_t * BN + 16 * TN * wn, c0 = first + 8 * lq;
        const bool whole = first + 16 * TN <= g.V;        // no column past the end
        #pragma unroll
        for (int i = 0; i < 4; i++) {
            const int m = m_t * BM + 64 * wm + 16 * i + lr;
            const int target = m < g.N ? g.targets[m] : -1;
            const int d = target - g.v0 - c0;             // the target's column from c0
            // this lane's part of the row has it (rare)
            const bool hit = target >= 0 && target - g.v0 < g.V && d >= 0 && d < 16 * TN && (d & 31) < 8;
            if constexpr (!GRAD) {
                float big = -INFINITY;
                if (!whole)
                    #pragma unroll
                    for (int t = 0; t < TN; t++)
                        #pragma unroll
                        for (int r = 0; r < 4; r++)
                            if (c0 + 32 * (t / 2) + 4 * (t & 1) + r >= g.V) acc[i][t][r] = -INFINITY;
                if (hit) {
                    float zt = 0.0f;
                    #pragma unroll
                    for (int t = 0; t < TN; t++)
                        #pragma unroll
                        for (int r = 0; r < 4; r++) zt = d == 32 * (t / 2) + 4 * (t & 1) + r ? acc[i][t][r] : zt;
                    g.hit[m] = zt;
                }
                #pragma unroll
                for (int t = 0; t < TN; t++)
                    #pragma unroll
                    for (int r = 0; r < 4; r++) big = fmaxf(big, acc[i][t][r]);
                big = fmaxf(big, kr_xor<16>(big));
                big = fmaxf(big, kr_xor<32>(big));
                // e^(z - big) as 2^(z log2 e - c); the rounding of c is taken back from the sum,
                // or, where it may be more than 1, there is none: z - big, then the product
                const float base = big == -INFINITY ? 0.0f : big;
                float c = base * kLog2e;
                float back = __builtin_amdgcn_exp2f(__builtin_fmaf(-base, kLog2e, c));
                if (fabsf(c) > 0x1p24f) {
                    #pragma unroll
                    for (int t = 0; t < TN; t++)
                        #pragma unroll
                        for (int r = 0; r < 4; r++) acc[i][t][r] -= base;
                    c = 0.0f;
                    back = 1.0f;
                }
                float sum = 0.0f;
                #pragma unroll
                for (int t = 0; t < TN; t++) {
                    float s = 0.0f;
                    #pragma unroll
                    for (int r = 0; r < 4; r++)
                        s += __builtin_amdgcn_exp2f(__builtin_fmaf(acc[i][t][r], kLog2e, -c));
                    sum += s;
                }
                sum += kr_xor<16>(sum);
                sum += kr_xor<32>(sum);
                if (m < g.N && lq == 0 && first < g.V)
                    g.part[(size_t)(n_t * WN + wn) * g.N + m] = float2{big, sum * back};
            } else {
                // f e^(z - lse) as 2^(z log2 e - c) with f's sign set behind it; beside a large
                // lse c's rounding would show (3e-4 of f at 8000): z - lse first
                float f = 0.0f, c = 0.0f;
                if (target != -1 && m < g.N) {
                    f = (unsigned)target < (unsigned)g.v_all ? g.dloss[m] * g.scale[0] : NAN;
                    const float lse = g.lse[m];
                    const bool first = fabsf(lse) > 32.0f;
                    c = (first ? 0.0f : lse * kLog2e) - __builtin_amdgcn_logf(fabsf(f));
                    if (first)
                        #pragma unroll
                        for (int t = 0; t < TN; t++)
                            #pragma unroll
                            for (int r = 0; r < 4; r++) acc[i][t][r] -= lse;
                }
                const float sign = f < 0.0f ? -1.0f : 1.0f;
                kr_half* out = g.G + (size_t)m * g.ldg + c0;
                #pragma unroll
                for (int p = 0; p < TN / 2; p++) {
                    float x[8];
                    #pragma unroll
                    for (int e = 0; e < 8; e++)
                        x[e] = sign * __builtin_amdgcn_exp2f(__builtin_fmaf(acc[i][2 * p + e / 4][e % 4], kLog2e, -c));
                    if (hit && (unsigned)(d - 32 * p) < 8u)
                        #pragma unroll
                        for (int e = 0; e < 8; e++)
                            if (d == 32 * p + e) {
                                x[e] -= f;
                                g.left[m] = f == 0.0f || g.G_low ? 0.0f : x[e] - (float)(kr_half)x[e];
                            }
                    if (!whole)
                        #pragma unroll
                        for (int e = 0; e < 8; e++)
                            if (c0 + 32 * p + e >= g.V) x[e] = 0.0f;
                    if (f == 0.0f)
                        #pragma unroll
                        for (int e = 0; e < 8; e++) x[e] = 0.0f;
                    kr_half8 v;
                    #pragma unroll
                    for (int e = 0; e < 8; e++) v[e] = (kr_half)x[e];
                    const bool on = m < g.rows && c0 + 32 * p < (int)g.ldg;
                    if (on) *reinterpret_cast<kr_half8*>(out + 32 * p) = v;
                    if (on && g.G_low) {
                        #pragma unroll
                        for (int e = 0; e < 8; e++) v[e] = (kr_half)(x[e] - (float)v[e]);
                        *reinterpret_cast<kr_half8*>(g.G_low + (out - g.G) + 32 * p) = v;
                    }
                }
            }
        }
        if (!has_next) break;
        vb += gridDim.x;
        m_t = nm_t;
        n_t = nn_t;
    }
}

// ---------------------------------------------------------------------------
// The forward pass of up to 16 rows: bound by W. Every wave walks 16-row blocks of W
// through an LDS ring of its own (steps of 64 k, whole lines, no barriers, 80 KB a CU in
// flight) beside x in LDS, and keeps a maximum and a sum per row. Measured on MI355X:
// 1 x 768 x 50277 17.7 us with the join's 4 (77 MB: 15.1 at a copy's rate). Limits: rows of
// one matrix instruction, and x in LDS. us, this kernel / the tiles: 1 x 768 x 50277 18.4 /
// 19.5, 8 rows 18.9 / 20.3, 16 19.4 / 21.0, of width 256 13.8 / 14.1, of 1536 33 / 31; over 4096
// columns 1 row 13.8 / 14.9, 16 14.0 / 14.8.
// ---------------------------------------------------------------------------
constexpr int kFewRows = 16, kFewC = 1536, kFewWaves = 8, kFewStages = 6;

__global__ void __launch_bounds__(64 * kFewWaves, 1) few_rows_kernel(LossArgs g) {
    __shared__ __attribute__((aligned(1024))) kr_half8 ring[kFewWaves * kFewStages * 128];
    __shared__ __attribute__((aligned(16))) kr_half8 xs[kFewRows * kFewC / 8];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int lr = lane & 15, lq = lane >> 4;
    const int KS = g.C / 64, units = g.C / 8, blocks = (g.V + 15) / 16;
    const int step = gridDim.x * kFewWaves, block0 = blockIdx.x + gridDim.x * wave;
    const unsigned ring_base = lds_address(ring) + (unsigned)(wave * kFewStages * 2048);
    int c_block = block0, c_ks = 0, c_stage = 0, ahead = 0;
    auto copy_step = [&]() {
        if (c_block >= blocks) return;
        const kr_half* wa = g.W + (long long)c_block * 16 * g.ldw;
        #pragma unroll
        for (int i = 0; i < 2; i++) {
            const int row = 8 * i + (lane >> 3), kc = (lane & 7) ^ ((row >> 1) & 7);
            const unsigned off = (unsigned)min(row, g.V - 1 - 16 * c_block) * (unsigned)(2 * g.ldw) +
                                 (unsigned)(16 * kc + 128 * c_ks);
            copy16(wa, off, ring_base + (unsigned)(c_stage * 2048 + 1024 * i));
        }
        ahead++;
        c_stage = c_stage + 1 == kFewStages ? 0 : c_stage + 1;
        if (++c_ks == KS) {
            c_ks = 0;
            c_block += step;
        }
    };
    #pragma unroll
    for (int i = 0; i < kFewStages - 1; i++) copy_step();
    for (int i = tid; i < kFewRows * units; i += 64 * kFewWaves) {
        const int n = i / units, u = i % units;
        kr_half8 v = {0, 0, 0, 0, 0, 0, 0, 0};
        if (n < g.N) v = *reinterpret_cast<const kr_half8*>(g.x + (size_t)n * g.ldx + 8 * u);
        xs[n * units + (u ^ (n & 7))] = v;
    }
    const int target = lr < g.N ? g.targets[lr] : -1;
    __syncthreads();
    float big = -INFINITY, sum = 0.0f;
    int stage = 0;
    for (int block = block0; block < blocks; block += step) {
        kr_float4 z = {0, 0, 0, 0};
        #pragma unroll 1
        for (int ks = 0; ks < KS; ks++) {
            if (ahead >= kFewStages - 1) wait_copies<(kFewStages - 2) * 2>();
            else wait_copies<0>();
            ahead--;
            const kr_half8* Ws = ring + (wave * kFewStages + stage) * 128;
            stage = stage + 1 == kFewStages ? 0 : stage + 1;
            #pragma unroll
            for (int kb = 0; kb < 2; kb++)
                z = __builtin_amdgcn_mfma_f32_16x16x32_f16(Ws[row_unit(lr, 4 * kb + lq)],
                                                           xs[lr * units + ((8 * ks + 4 * kb + lq) ^ (lr & 7))], z, 0,
                                                           0, 0);
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");    // the stage is read
            copy_step();
        }
        const int v0 = 16 * block + 4 * lq, d = target - v0;
        float to = big;
        #pragma unroll
        for (int r = 0; r < 4; r++) {
            if (d == r && v0 + r < g.V) g.hit[lr] = z[r];
            if (v0 + r >= g.V) z[r] = -INFINITY;
            to = fmaxf(to, z[r]);
        }
        const float base = to == -INFINITY ? 0.0f : to;
        sum *= __builtin_amdgcn_exp2f((big - base) * kLog2e);
        #pragma unroll
        for (int r = 0; r < 4; r++) sum += __builtin_amdgcn_exp2f((z[r] - base) * kLog2e);
        big = to;
    }
    // the 4 x 8 parts of a row
    __syncthreads();
    float2* parts = reinterpret_cast<float2*>(xs);
    parts[(4 * wave + lq) * 16 + lr] = float2{big, sum};
    __syncthreads();
    if (tid >= g.N) return;
    big = -INFINITY;
    for (int p = 0; p < 4 * kFewWaves; p++) big = fmaxf(big, parts[p * 16 + tid].x);
    const float base = big == -INFINITY ? 0.0f : big;
    sum = 0.0f;
    for (int p = 0; p < 4 * kFewWaves; p++)
        sum += parts[p * 16 + tid].y * __builtin_amdgcn_exp2f((parts[p * 16 + tid].x - base) * kLog2e);
    g.part[(size_t)blockIdx.x * g.N + tid] = float2{big, sum};
}

// Parts of a row -> lse and loss; ROWS rows x 256 / ROWS parts at a time.
template <int ROWS>
__global__ void __launch_bounds__(256) loss_join_kernel(const float2* part, const float* hit, int N, int parts,
                                                        int V, const int32_t* targets, float* loss, float* lse) {
    constexpr int LANES = 256 / ROWS;
    __shared__ float big_of[LANES][ROWS], sum_of[LANES][ROWS];
    const int r = threadIdx.x % ROWS, p0 = threadIdx.x / ROWS;
    const int m = blockIdx.x * ROWS + r;
    float big = -INFINITY, sum = 0.0f;
    constexpr int kAhead = 8;             // or every step waits for memory
    if (m < N)
        for (int p = p0; p < parts; p += kAhead * LANES) {
            float2 v[kAhead];
            #pragma unroll
            for (int i = 0; i < kAhead; i++)
                v[i] = p + i * LANES < parts ? part[(size_t)(p + i * LANES) * N + m] : float2{-INFINITY, 0.0f};
            float to = big;
            #pragma unroll
            for (int i = 0; i < kAhead; i++) to = fmaxf(to, v[i].x);
            const float base = to == -INFINITY ? 0.0f : to;
            sum *= __builtin_amdgcn_exp2f((big - base) * kLog2e);
            #pragma unroll
            for (int i = 0; i < kAhead; i++) sum += v[i].y * __builtin_amdgcn_exp2f((v[i].x - base) * kLog2e);
            big = to;
        }
    big_of[p0][r] = big;
    sum_of[p0][r] = sum;
    __syncthreads();
    if (ROWS == 1) {                      // 256 parts: first to 4 waves', then together
        const float most = kr_wave_reduce(big, [](float a, float b) { return fmaxf(a, b); });
        const float base = most == -INFINITY ? 0.0f : most;
        sum = kr_wave_reduce(sum * __builtin_amdgcn_exp2f((big - base) * kLog2e), [](float a, float b) { return a + b; });
        __syncthreads();
        if ((threadIdx.x & 63) == 0) {
            big_of[threadIdx.x >> 6][0] = most;
            sum_of[threadIdx.x >> 6][0] = sum;
        }
        __syncthreads();
    }
    if (threadIdx.x >= ROWS || m >= N) return;
    constexpr int LEFT = ROWS == 1 ? 4 : LANES;
    big = -INFINITY;
    for (int p = 0; p < LEFT; p++) big = fmaxf(big, big_of[p][r]);
    const float base = big == -INFINITY ? 0.0f : big;
    sum = 0.0f;
    for (int p = 0; p < LEFT; p++) sum += sum_of[p][r] * __builtin_amdgcn_exp2f((big_of[p][r] - base) * kLog2e);
    const float ln_sum = __builtin_amdgcn_logf(sum) * kLn2;
    const int target = targets[m];
    lse[m] = base + ln_sum;
    loss[m] = target == -1 ? 0.0f : (unsigned)target < (unsigned)V ? (base - hit[m]) + ln_sum : NAN;
}

// ---------------------------------------------------------------------------
// Backward: the power of two of dz (the last workgroup), and x with the rows that have
// no gradient as zeros (whatever they hold), rounded up to 64 rows.
// ---------------------------------------------------------------------------
__global__ void __launch_bounds__(1024) grad_prepare_kernel(const kr_half* x, long long ldx, int N, int C, int rows,
                                                            const int32_t* targets, const float* dloss,
                                                            float* scale, kr_half* out) {
    __shared__ float part[16];
    if (blockIdx.x + 1 < gridDim.x) {
        const int per = C / 8;
        const long long at = (long long)blockIdx.x * 1024 + threadIdx.x;
        if (at >= (long long)rows * per) return;
        const int m = (int)(at / per), c = 8 * (int)(at % per);
        kr_half8 v = {0, 0, 0, 0, 0, 0, 0, 0};
        if (m < N && targets[m] != -1 && dloss[m] != 0.0f)
            v = *reinterpret_cast<const kr_half8*>(x + (size_t)m * ldx + c);
        *reinterpret_cast<kr_half8*>(out + (size_t)m * C + c) = v;
        return;
    }
    float big = 0.0f;
    for (int i0 = threadIdx.x; i0 < N; i0 += 8 * 1024) {
        float a[8];
        int t[8];
        #pragma unroll
        for (int j = 0; j < 8; j++) {
            const int i = min(i0 + 1024 * j, N - 1);
            a[j] = fabsf(dloss[i]);
            t[j] = targets[i];
        }
        #pragma unroll
        for (int j = 0; j < 8; j++)
            if (t[j] != -1 && a[j] < INFINITY) big = fmaxf(big, a[j]);
    }
    big = kr_wave_reduce(big, [](float a, float b) { return fmaxf(a, b); });
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = big;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int i = 0; i < 16; i++) big = fmaxf(big, part[i]);
        int e = (int)(__float_as_uint(big) >> 23);        // 2^(e - 127) <= big
        e = e < 15 ? 15 : e;
        scale[0] = __uint_as_float((uint32_t)(268 - e) << 23);     // 2^(141 - e)
        scale[1] = __uint_as_float((uint32_t)(e - 14) << 23);
    }
}

// ---------------------------------------------------------------------------
// dW += dz' x and dx += dz W of one piece, in tiles of (64 WM) x (16 TN WN), a wave for
// each 64 x 16 TN, steps of 64 k through two stages. Operands whose rows lie across k
// (W and x as B, dz' as A) are staged as they lie, 64 k x the tile's columns, and
// read by the LDS's transposing reads: 16 lanes get 4 k of 16 columns.
// Bound: copies (one step ahead) and the last round of workgroups: dW's tiles of a piece
// take all N rows each, dx's splits fill up behind them. Measured on MI355X, a piece of
// 10240 columns of 8192 x 768 x 50277: 283 us for both products (0.90 PF/s; a library's of
// these sizes 0.77 dW, 1.04 dx); steps of 32 k, three ahead, 292. Pieces: a call's workspace
// is what keeps dz at 176 MB, not its time, which goes by how the rounds of workgroups of a
// piece come out. us, 176 / 352 / 420 / 880 MB: 8192 x 768 x 50277 2060 / 2226 / 2004 / 1993, 512
// wide 1538 / 1647 / 1680 / 1659, 4096 x 768 1245 / 1092 / 1029 / 1038, 16384 x 768 4758 / 3885 /
// 4007 / 3855, 30000 x 256 x 4096 360 / 331 / 332 / 331.
// ---------------------------------------------------------------------------
struct ProdArgs {
    const kr_half* G;                 // [rows][ldg]
    long long ldg;
    int parts;                        // 2: and what fp16 left of it, behind
    const kr_half* x;                 // [rows][C]
    const kr_half* W;                 // [V, C] of the piece
    long long ldw;
    const float* scale;
    const kr_half* W_all;             // [V, C]
    const int32_t* targets;
    const float* left;
    int v_all;
    float* dx_part;                   // [dx_splits][rows][C], if not direct
    float* dw_part;                   // [dw_splits][V][C], if not direct
    void* dx;                         // [N][C], direct: one split, one piece
    void* dW;                         // [V][C] of the piece, direct: one split
    int f32;                          // their type
    int N, rows, C, V, first;         // first: dx_part is written, not added to
    int v0;                           // the piece's first column
    int dx_splits, dw_splits, dx_direct;
    int dw_run;                       // column tiles that an item of dW takes in turn
    int dw_items, dx_items;
};

// Columns that lie across k, in an LDS tile of COLS of them: place, in bytes, of this
// lane's 4 columns of a 16-column tile for k = 8 (l / 16) + (l % 16) / 4, with the tile
// XORed by a value of k's bits 0, 1 and 3, so that the 32 lanes of half a read are on
// different banks.
template <int COLS>
__device__ __forceinline__ unsigned across(int tile, int lane) {
    const int lr = lane & 15, lq = lane >> 4;
    const int sw = (lr >> 2) | ((lq & 1) << 2);
    return (unsigned)((8 * lq + (lr >> 2)) * 2 * COLS + 32 * (tile ^ sw) + 8 * (lr & 3));
}
template <int COLS>
__device__ __forceinline__ kr_half8 read_across(unsigned at) {
    typedef kr_half half4v __attribute__((ext_vector_type(4)));
    const half4v lo = __builtin_bit_cast(half4v, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4*)(uintptr_t)at));
    const half4v hi = __builtin_bit_cast(
        half4v, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4*)(uintptr_t)(at + 8 * COLS)));
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
}

// Copies of one step of an operand, 64 k x COLS, by half of the workgroup's waves.
template <int COLS, int COPIES>
__device__ __forceinline__ void copy_across(const kr_half* base, long long ld, int last, int cols, unsigned to,
                                            int part, int lane) {
    constexpr int PER = 512 / COLS, LANES = 64 / PER;     // rows of a copy, lanes of a row
    base = shared_by_lanes(base);
    #pragma unroll
    for (int i = 0; i < COPIES; i++) {
        const int k = PER * (part * COPIES + i) + lane / LANES;
        const int sw = 2 * ((k & 3) | ((k >> 1) & 4));
        const int col = 8 * ((lane % LANES) ^ sw);
        const unsigned off = (unsigned)min(k, last) * (unsigned)(2 * ld) + (unsigned)(col < cols ? 2 * col : 0);
        copy16(base, off, to + 1024u * (unsigned)(part * COPIES + i));
    }
}

// What fp16 left of the target's dz (one value, but of most of a row's dx: 4.2e-4 of it
// without this, 2.2e-4 with) times its row of W; its row of x goes into dW (TargetRows).
struct TargetRest {
    const kr_half* w;
    float left;
    __device__ TargetRest(const kr_half* W, long long ldw, int V, const int32_t* targets, const float* rest, int m) {
        const int t = targets[m];
        const bool on = (unsigned)t < (unsigned)V;
        w = W + (on ? (size_t)t * ldw : 0);
        left = on ? rest[m] : 0.0f;
    }
    __device__ kr_half4 row(int n) const { return *reinterpret_cast<const kr_half4*>(w + n); }
    __device__ kr_float4 times(kr_half4 x) const {       // 0 where there is none, whatever W has
        kr_float4 v;
        #pragma unroll
        for (int r = 0; r < 4; r++) v[r] = left == 0.0f ? 0.0f : left * (float)x[r];
        return v;
    }
};

__device__ __forceinline__ void store_out(void* out, size_t at, kr_float4 v, int f32) {
    if (f32) *reinterpret_cast<kr_float4*>(static_cast<float*>(out) + at) = v;
    else
        *reinterpret_cast<kr_half4*>(static_cast<kr_half*>(out) + at) =
            kr_half4{kr_f16(v[0]), kr_f16(v[1]), kr_f16(v[2]), kr_f16(v[3])};
}

// The rows n of a range whose target is one of `columns` from v0, and what fp16 left of
// its dz, in their order, some kHits at a time: a tile of dW takes them after its other
// rows, 64 a step. Of dW's 2-norm the rest is 2.1e-4 on average, as the rounding of an
// fp16 output is, and 3.9e-4 where all dloss are just above a power of two; without it
// 6e-5 is left, the other dz's. All waves look through all rows and write the same list, so
// that none waits for another. Measured on MI355X, gradients with / without: 8192 x 768 x 50277
// 2069 / 2053 us, 20000 x 256 x 256 (half of all rows in every tile) 44.8 / 41.8, 97 x 1024 x
// 50277 122.6 / 112.6 (three barriers and a step in a quarter of the tiles, which have two
// steps without).
constexpr int kHits = 1024, kLooked = 8 * 64;
struct TargetRows {
    int2* list;                       // n; column | fp16 rest << 16
    int end, v0, columns;
    int at, count;                    // the next row to look at, entries of the list

    __device__ void fill(const int32_t* targets, const float* left, int lane) {
        count = 0;
        while (at < end && count <= kHits - kLooked) {
            int column[8];
            float rest[8];
            #pragma unroll
            for (int j = 0; j < 8; j++) {
                const int n = min(at + 64 * j + lane, end - 1);
                column[j] = targets[n] - v0;
                rest[j] = left[n];
            }
            #pragma unroll
            for (int j = 0; j < 8; j++) {
                const int n = at + 64 * j + lane;
                const bool on = n < end && (unsigned)column[j] < (unsigned)columns && rest[j] != 0.0f;
                const uint64_t all = __ballot(on);
                if (on)
                    list[count + __popcll(all & ((1ull << lane) - 1))] =
                        int2{n, column[j] | (int)__builtin_bit_cast(uint16_t, (kr_half)rest[j]) << 16};
                count += __popcll(all);
            }
            at += kLooked;
        }
    }
};

// A stage of 64 of them: A zeros but for the rests, B their rows of x. Past the list's end
// the last row again, against zeros.
template <int BM, int BN, int WAVES>
__device__ __forceinline__ void target_step(const TargetRows& r, int e0, const kr_half* x, int ldx, int cols,
                                            kr_half8* stage, unsigned at, int tid, int wave, int lane) {
    constexpr int PER = 512 / BN, LANES = 64 / PER, COPIES = BN / 8 / WAVES;
    auto swap = [](int k) { return 2 * ((k & 3) | ((k >> 1) & 4)); };       // as copy_across has it
    #pragma unroll
    for (int i = 0; i < COPIES; i++) {
        const int k = PER * (wave * COPIES + i) + lane / LANES;
        const int col = 8 * ((lane % LANES) ^ swap(k));
        const kr_half* src = x + (size_t)r.list[min(e0 + k, r.count - 1)].x * ldx + (col < cols ? col : 0);
        kr_copy16(src, (unsigned)__builtin_amdgcn_readfirstlane((int)(at + BM * 128u + 1024u * (wave * COPIES + i))));
    }
    #pragma unroll
    for (int i = 0; i < BM / 8 / WAVES; i++) stage[64 * WAVES * i + tid] = kr_half8{0, 0, 0, 0, 0, 0, 0, 0};
    __syncthreads();
    if (tid < 64 && e0 + tid < r.count) {
        const int v = r.list[e0 + tid].y, column = v & 0xffff;
        reinterpret_cast<uint16_t*>(stage + tid * (BM / 8) + ((column / 8) ^ swap(tid)))[column % 8] = (uint16_t)(v >> 16);
    }
    wait_copies<0>();
    __syncthreads();
}

template <int WM, int WN, int TN, bool DW>
__device__ __forceinline__ void product_tile(const ProdArgs& g, kr_half8* ring, int2* hits, int item) {
    constexpr int BM = 64 * WM, BN = 16 * TN * WN, WAVES = WM * WN;
    static_assert(BM == BN, "half of the waves copy each operand");
    constexpr int COPIES = BM / 8 / (WAVES / 2), STAGE = (BM + BN) * 8;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave / WN, wn = wave % WN;
    const int lr = lane & 15, lq = lane >> 4;
    const int gx = (g.C + BN - 1) / BN;
    const int splits = DW ? g.dw_splits : g.dx_splits;
    const int runs = DW ? (gx + g.dw_run - 1) / g.dw_run : gx;
    const int n_first = item % runs * (DW ? g.dw_run : 1), n_last = DW ? min(n_first + g.dw_run, gx) : n_first + 1;
    const int m_t = item / runs / splits, split = item / runs % splits;
    const int M = DW ? g.V : g.rows;
    const int more = g.parts - 1;         // a second step for every 64 k, with the low parts
    const int steps = (DW ? g.rows / 64 : (g.V + 63) / 64) << more;
    const int ks0 = (int)((long long)steps * split / splits), ks1 = (int)((long long)steps * (split + 1) / splits);
    const unsigned ring_base = lds_address(ring);
    const int m0 = m_t * BM;
    // A: dW reads G across (columns m0.., always inside ldg), dx along
    const kr_half* a_base = DW ? g.G + m0 : g.G + (size_t)m0 * g.ldg;
    const kr_half* b_base = DW ? g.x : g.W;
    const long long ldb = DW ? g.C : g.ldw;
    auto issue = [&](int n_t, int step, int q) {
        const unsigned so = ring_base + (unsigned)((q & 1) * STAGE * 16);
        const int n0 = n_t * BN, ks = step >> more;
        const kr_half* a = a_base + (step & more ? (size_t)g.rows * g.ldg : 0);
        if (wave >= WAVES / 2) {
            // B's k past the piece: the last row, against zeros of G
            copy_across<BN, COPIES>(b_base + n0 + (long long)ks * 64 * ldb, ldb, DW ? 63 : g.V - 1 - 64 * ks, g.C - n0,
                                    so + BM * 128, wave - WAVES / 2, lane);
        } else if (DW) {
            copy_across<BM, COPIES>(a + (long long)ks * 64 * g.ldg, g.ldg, 63, (int)g.ldg - m0, so, wave, lane);
        } else {
            #pragma unroll
            for (int i = 0; i < COPIES; i++) {
                const int row = 8 * (wave * COPIES + i) + (lane >> 3);
                const int kc = (lane & 7) ^ ((row >> 1) & 7);
                const unsigned off = (unsigned)min(row, M - 1 - m0) * (unsigned)(2 * g.ldg) +
                                     (unsigned)(16 * kc + 128 * ks);
                copy16(a, off, so + 1024u * (unsigned)(wave * COPIES + i));
            }
        }
    };
    unsigned a_at[4], b_at[TN];
    #pragma unroll
    for (int i = 0; i < 4; i++) a_at[i] = across<BM>(4 * wm + i, lane);
    #pragma unroll
    for (int t = 0; t < TN; t++) b_at[t] = across<BN>(TN * wn + t, lane) + BM * 128u;
    const float down = g.scale[1];
    const bool direct = DW ? splits == 1 : g.dx_direct != 0;
    const int m_end = !DW && direct ? g.N : M;
    int q = 0;
    // a short last piece has fewer steps than dx's splits: one without steps only adds zeros
    if (ks0 < ks1) issue(n_first, ks0, 0);
    // with low parts nothing is left of the targets' dz
    TargetRows rows{hits, more ? 0 : min(64 * ks1, g.N), g.v0 + m0, min(BM, g.V - m0), 64 * ks0, 0};
    if (DW) rows.fill(g.targets, g.left, lane);
    for (int n_t = n_first; n_t < n_last; n_t++) {
        kr_float4 acc[4][TN];
        #pragma unroll
        for (int i = 0; i < 4; i++)
            #pragma unroll
            for (int t = 0; t < TN; t++) acc[i][t] = kr_float4{0, 0, 0, 0};
        auto multiply = [&](int stage) {
            const kr_half8* As = ring + stage * STAGE;
            const unsigned so = ring_base + (unsigned)(stage * STAGE * 16);
            #pragma unroll
            for (int kb = 0; kb < 2; kb++) {
                kr_half8 a[4];
                #pragma unroll
                for (int i = 0; i < 4; i++)
                    a[i] = DW ? read_across<BM>(so + a_at[i] + 64u * BM * kb)
                              : As[row_unit(64 * wm + 16 * i + lr, 4 * kb + lq)];
                #pragma unroll
                for (int th = 0; th < TN / 4; th++) {
                    __builtin_amdgcn_sched_barrier(0);
                    kr_half8 b[4];
                    #pragma unroll
                    for (int t = 0; t < 4; t++) b[t] = read_across<BN>(so + b_at[4 * th + t] + 64u * BN * kb);
                    __builtin_amdgcn_sched_barrier(0);
                    #pragma unroll
                    for (int i = 0; i < 4; i++)
                        #pragma unroll
                        for (int t = 0; t < 4; t++)
                            acc[i][4 * th + t] =
                                __builtin_amdgcn_mfma_f32_16x16x32_f16(b[t], a[i], acc[i][4 * th + t], 0, 0, 0);
                }
            }
        };
        #pragma unroll 1
        for (int ks = ks0; ks < ks1; ks++, q++) {
            wait_copies<0>();
            __syncthreads();   // every wave's copies are in; the step before is read
            if (ks + 1 < ks1) issue(n_t, ks + 1, q + 1);
            else if (n_t + 1 < n_last) issue(n_t + 1, ks0, q + 1);
            multiply(q & 1);
        }
        if constexpr (DW) {
            // the targets' rests, 64 rows of x a step, in the stage read last
            const int stage = (q + 1) & 1, n0 = n_t * BN;
            while (true) {                    // a run of column tiles has one list (dw_run)
                #pragma unroll 1
                for (int e0 = 0; e0 < rows.count; e0 += 64) {
                    __syncthreads();   // the stage is read
                    target_step<BM, BN, WAVES>(rows, e0, g.x + n0, g.C, g.C - n0, ring + stage * STAGE,
                                               ring_base + (unsigned)(stage * STAGE * 16), tid, wave, lane);
                    multiply(stage);
                }
                if (rows.at >= rows.end) break;
                rows.fill(g.targets, g.left, lane);
            }
        }
        #pragma unroll
        for (int i = 0; i < 4; i++) {
            const int m = m0 + 64 * wm + 16 * i + lr, c0 = n_t * BN + 16 * TN * wn + 4 * lq;
            if (m >= m_end) continue;
            if (!DW && direct) {
                const TargetRest rest(g.W_all, g.ldw, g.v_all, g.targets, g.left, m);
                kr_half4 w[TN];
                #pragma unroll
                for (int t = 0; t < TN; t++) w[t] = rest.row(c0 + 16 * t < g.C ? c0 + 16 * t : 0);
                #pragma unroll
                for (int t = 0; t < TN; t++)
                    if (c0 + 16 * t < g.C)
                        store_out(g.dx, (size_t)m * g.C + c0 + 16 * t, (acc[i][t] + rest.times(w[t])) * down, g.f32);
                continue;
            }
            #pragma unroll
            for (int t = 0; t < TN; t++) {
                const int n = c0 + 16 * t;
                if (n >= g.C) continue;
                kr_float4 v = acc[i][t];
                if (direct) {
                    store_out(g.dW, (size_t)m * g.C + n, v * down, g.f32);
                } else {
                    float* part = DW ? g.dw_part : g.dx_part;
                    kr_float4* o = reinterpret_cast<kr_float4*>(part + ((size_t)split * M + m) * g.C + n);
                    if (!DW && !g.first) v += *o;
                    *o = v;
                }
            }
        }
    }
}

// Item of workgroup b: an eighth of the items in order for each XCD.
__device__ __forceinline__ int item_of(int b, int items) {
    const int per = (items + 7) / 8, full = items % 8 ? items % 8 : 8;
    const int xcd = b & 7, i = b >> 3;
    return xcd < full ? xcd * per + i : full * per + (xcd - full) * (per - 1) + i;
}

template <int WM, int WN, int TN>
__global__ void __launch_bounds__(64 * WM * WN, WM * WN >= 8 ? 1 : 2) grad_products_kernel(ProdArgs g) {
    __shared__ __attribute__((aligned(1024))) kr_half8 ring[2 * (64 * WM + 16 * TN * WN) * 8];
    __shared__ int2 hits[kHits];
    // dW's items before dx's
    const int b = blockIdx.x;
    if (b < g.dw_items) product_tile<WM, WN, TN, true>(g, ring, hits, item_of(b, g.dw_items));
    else product_tile<WM, WN, TN, false>(g, ring, hits, item_of(b - g.dw_items, g.dx_items));
}

// Sum of the splits of n outputs, in their order; of dx (W not null), with the targets' rest.
__global__ void __launch_bounds__(256) grad_sum_kernel(const float* part, long long stride, int splits, long long n,
                                                       const float* scale, int f32, void* out, const kr_half* W,
                                                       long long ldw, int V, const int32_t* targets,
                                                       const float* left, int C) {
    const long long at = 4 * ((long long)blockIdx.x * 256 + threadIdx.x);
    if (at >= n) return;
    kr_float4 v = {0, 0, 0, 0};
    constexpr int kAhead = 8;             // or every split waits for memory
    for (int s = 0; s < splits; s += kAhead) {
        kr_float4 x[kAhead];
        #pragma unroll
        for (int i = 0; i < kAhead; i++)
            x[i] = s + i < splits ? *reinterpret_cast<const kr_float4*>(part + (s + i) * stride + at) : kr_float4{0, 0, 0, 0};
        #pragma unroll
        for (int i = 0; i < kAhead; i++) v += x[i];
    }
    if (W) {
        const TargetRest rest(W, ldw, V, targets, left, (int)(at / C));
        v += rest.times(rest.row((int)(at % C)));
    }
    store_out(out, at, v * scale[1], f32);
}

template <int WM, int WN, int TN, bool GRAD>
int launch_logits(const LossArgs& g, hipStream_t s) {
    constexpr int BM = 64 * WM, BN = 16 * TN * WN;
    const int gy = ((GRAD ? g.rows : g.N) + BM - 1) / BM, gx = (g.V + BN - 1) / BN;
    const long long tiles = (long long)gx * gy;
    const int n_virtual = (int)((tiles + 7) / 8 * 8);
    const int at_once = 256 * (WM * WN >= 8 ? 1 : 2);
    const int grid = n_virtual < at_once ? n_virtual : at_once;
    // about 1.25 MB of x to a group of row tiles, as an L2 holds beside W's
    const int group_m = (int)std::min<long long>(8, std::max<long long>(1, (5ll << 18) / (BM * 2ll * g.C)));
    logits_kernel<WM, WN, TN, GRAD><<<grid, 64 * WM * WN, 0, s>>>(g, n_virtual, group_m);
    KR_LAUNCHED();
    return KR_OK;
}

// Which tiles. us, 128 x 128 / 256 x 256, width 768: losses over 50277 columns of 128
// rows 23 / 32, 256 39 / 32, 1024 104 / 104, 4096 372 / 314; over 4096 columns of 2048 rows
// (128 large tiles) 20 / 29, 8192 64 / 56. Gradients, of which dz is in them: over 50277
// columns 128 rows 91 / 101, 256 141 / 131, 1024 336 / 334, 8192 2186 / 2056; over 4096
// columns 2048 rows 80 / 88, 8192 219 / 211.
bool big_tiles(int N, int V) {
    return N > 128 && (long long)((N + 255) / 256) * ((V + 255) / 256) >= 192;
}

template <bool GRAD>
int logits(const LossArgs& g, bool big, hipStream_t s) {
    return big ? launch_logits<4, 2, 8, GRAD>(g, s) : launch_logits<2, 2, 4, GRAD>(g, s);
}

// Forward: parts of a row, and their count.
bool few_rows(int N, int C) { return N <= kFewRows && C <= kFewC; }
int loss_parts(int N, int C, int V) {
    if (few_rows(N, C)) return std::min(256, (V + 16 * kFewWaves - 1) / (16 * kFewWaves));
    return big_tiles(N, V) ? (V + 127) / 128 : (V + 63) / 64;
}

bool shape_ok(int N, int C, int V) {
    return N >= 0 && N <= 1 << 24 && C >= 64 && C % 64 == 0 && C <= 1 << 14 && V >= 1 && V <= 1 << 24 &&
           (long long)N * V <= 1ll << 44;             // a launch's tiles stay below 2^31
}
// Backward, also what a thread for four values of dx or dW (and one for eight of x) can be
// launched for, 2^32.
bool grad_shape_ok(int N, int C, int V) {
    return shape_ok(N, C, V) && (long long)N * C <= 1ll << 33 && (long long)V * C <= 1ll << 33;
}
constexpr int kLossRows = 1 << 16;                    // of a forward launch: bounds its parts

size_t up256(size_t n) { return (n + 255) / 256 * 256; }

// How a backward call is cut: pieces of the vocabulary whose dz takes at most
// 176 MB, and the products' splits.
struct GradPlan {
    int rows, piece, pieces, dx_splits, dw_splits, dw_run;
    bool big, big_products, dx_direct;
    size_t left, x, G, dx_part, dw_part, total;             // offsets in the workspace
};

GradPlan grad_plan(int N, int C, int V, bool dx, bool dw, int parts) {
    GradPlan p{};
    p.rows = (N + 63) / 64 * 64;
    const long long most = std::max<long long>(256, (88ll << 20) / parts / p.rows / 256 * 256);
    p.pieces = (int)((V + most - 1) / most);
    p.piece = ((V + p.pieces - 1) / p.pieces + 255) / 256 * 256;
    p.pieces = (V + p.piece - 1) / p.piece;
    p.big = big_tiles(N, V);
    // us for gradients, 128 x 128 / 256 x 256 tiles in the products: 8192 x 768 x 50277 2167 /
    // 2061, 512 wide 1503 / 1711, 4096 x 256 wide 532 / 603, 16384 x 768 x 16384 (66 tiles of dW
    // a piece) 1507 / 1838, 4096 x 1024 x 4096 (64) 135 / 187
    p.big_products = p.big && C > 512 && (p.piece / 256) * ((C + 255) / 256) >= 100;
    const int tile = p.big_products ? 256 : 128, slots = p.big_products ? 256 : 512;
    const int gx = (C + tile - 1) / tile, dx_steps = p.piece / 64 * parts, dw_steps = p.rows / 64 * parts;
    const long long dx_tiles = (long long)(p.rows + tile - 1) / tile * gx, dw_tiles = (long long)p.piece / tile * gx;
    const long long total = (dx ? dx_tiles * dx_steps : 0) + (dw ? dw_tiles * dw_steps : 0);
    const long long each = std::max<long long>(8, total / (3 * slots));
    p.dx_splits = (int)std::max<long long>(1, std::min<long long>(64, dx_steps / each));
    p.dw_splits = dw_tiles >= slots / 4 ? 1 : (int)std::max<long long>(1, std::min<long long>(64, dw_steps / each));
    p.dw_run = p.rows <= kLooked && p.dw_splits == 1 ? gx : 1;
    p.dx_direct = p.dx_splits == 1 && p.pieces == 1;
    size_t at = 256;                                  // the scale
    p.left = at;
    at += up256((size_t)p.rows * 4);
    p.x = at;
    at += up256((size_t)p.rows * C * 2);
    p.G = at;
    at += up256((size_t)p.rows * p.piece * 2 * parts);
    p.dx_part = at;
    if (dx && !p.dx_direct) at += up256((size_t)p.dx_splits * p.rows * C * 4);
    p.dw_part = at;
    if (dw && p.dw_splits > 1) at += up256((size_t)p.dw_splits * std::min(V, p.piece) * C * 4);
    p.total = at;
    return p;
}

}  // namespace

extern "C" {

size_t kr_head_loss_workspace_bytes(int N, int C, int V) {
    if (!shape_ok(N, C, V) || N == 0) return 0;
    const int rows = std::min(N, kLossRows), last = (N - 1) % kLossRows + 1;
    const size_t parts = std::max((size_t)loss_parts(rows, C, V) * rows, (size_t)loss_parts(last, C, V) * last);
    return up256((size_t)rows * 4) + parts * sizeof(float2);
}

int kr_head_loss(const uint16_t* x, long long ldx, int N, int C, const uint16_t* W, long long ldw, int V,
                 const int32_t* targets, float* loss, float* lse, void* ws, size_t ws_bytes, void* stream) {
    KR_REQUIRE(shape_ok(N, C, V), "kr_head_loss: bad shape N=%d C=%d V=%d (C a multiple of 64 up to 16384, N and V up to 2^24, N * V up to 2^44)",
               N, C, V);
    KR_REQUIRE(ldx >= C && ldw >= C && (ldx | ldw) % 8 == 0 && (ldx | ldw) < 1 << 21,
               "kr_head_loss: row strides must be multiples of 8, at least C = %d and below 2^21", C);
    if (N == 0) return KR_OK;
    KR_REQUIRE(x && W && targets && loss && lse, "kr_head_loss: null pointer");
    KR_REQUIRE((((uintptr_t)x | (uintptr_t)W) & 15) == 0, "kr_head_loss: x and W must be 16-byte aligned");
    const size_t need = kr_head_loss_workspace_bytes(N, C, V);
    KR_REQUIRE(ws && ws_bytes >= need && ((uintptr_t)ws & 255) == 0,
               "kr_head_loss: workspace of %zu bytes, %zu needed (256-byte aligned)", ws_bytes, need);
    LossArgs g{};
    g.W = reinterpret_cast<const kr_half*>(W);
    g.ldx = ldx;
    g.ldw = ldw;
    g.hit = static_cast<float*>(ws);
    g.part = reinterpret_cast<float2*>(static_cast<char*>(ws) + up256((size_t)std::min(N, kLossRows) * 4));
    g.C = C;
    g.V = g.v_all = V;
    const hipStream_t s = kr_stream(stream);
    for (int r0 = 0; r0 < N; r0 += kLossRows) {
        const int n = std::min(N - r0, kLossRows), parts = loss_parts(n, C, V);
        g.x = reinterpret_cast<const kr_half*>(x) + (size_t)r0 * ldx;
        g.targets = targets + r0;
        g.N = n;
        if (few_rows(n, C)) {
            few_rows_kernel<<<parts, 64 * kFewWaves, 0, s>>>(g);
            KR_LAUNCHED();
        } else {
            const int rc = logits<false>(g, big_tiles(n, V), s);
            if (rc != KR_OK) return rc;
        }
        if (n <= 256)
            loss_join_kernel<1><<<n, 256, 0, s>>>(g.part, g.hit, n, parts, V, g.targets, loss + r0, lse + r0);
        else
            loss_join_kernel<16><<<(n + 15) / 16, 256, 0, s>>>(g.part, g.hit, n, parts, V, g.targets, loss + r0, lse + r0);
        KR_LAUNCHED();
    }
    return KR_OK;
}

size_t kr_head_loss_backward_workspace_bytes(int N, int C, int V, int dx, int dw) {
    if (!grad_shape_ok(N, C, V) || N == 0) return 0;
    return std::max(grad_plan(N, C, V, dx != 0, dw != 0, 1).total, grad_plan(N, C, V, dx != 0, dw != 0, 2).total);
}

int kr_head_loss_backward(const uint16_t* x, long long ldx, int N, int C, const uint16_t* W, long long ldw, int V,
                          const int32_t* targets, const float* lse, const float* dloss, int out_f32, void* dx,
                          void* dW, void* ws, size_t ws_bytes, void* stream) {
    KR_REQUIRE(grad_shape_ok(N, C, V),
               "kr_head_loss_backward: bad shape N=%d C=%d V=%d (C a multiple of 64 up to 16384, N and V up to 2^24, N * V up to 2^44, N * C and V * C up to 2^33)",
               N, C, V);
    KR_REQUIRE(N >= 1, "kr_head_loss_backward: no rows");
    KR_REQUIRE(ldx >= C && ldw >= C && (ldx | ldw) % 8 == 0 && (ldx | ldw) < 1 << 21,
               "kr_head_loss_backward: row strides must be multiples of 8, at least C = %d and below 2^21", C);
    KR_REQUIRE(x && W && targets && lse && dloss && (dx || dW), "kr_head_loss_backward: null pointer");
    KR_REQUIRE((((uintptr_t)x | (uintptr_t)W | (uintptr_t)dx | (uintptr_t)dW) & 15) == 0,
               "kr_head_loss_backward: x, W, dx and dW must be 16-byte aligned");
    const int parts = out_f32 ? 2 : 1;
    const GradPlan p = grad_plan(N, C, V, dx != nullptr, dW != nullptr, parts);
    const size_t need = kr_head_loss_backward_workspace_bytes(N, C, V, dx != nullptr, dW != nullptr);
    KR_REQUIRE(ws && ws_bytes >= need && ((uintptr_t)ws & 255) == 0,
               "kr_head_loss_backward: workspace of %zu bytes, %zu needed (256-byte aligned)", ws_bytes, need);
    char* base = static_cast<char*>(ws);
    float* scale = reinterpret_cast<float*>(base);
    kr_half* live = reinterpret_cast<kr_half*>(base + p.x);
    const kr_half* xh = reinterpret_cast<const kr_half*>(x);
    const hipStream_t s = kr_stream(stream);
    const long long units = dW ? (long long)p.rows * (C / 8) : 0;
    grad_prepare_kernel<<<(unsigned)((units + 1023) / 1024 + 1), 1024, 0, s>>>(xh, ldx, N, C, p.rows, targets, dloss,
                                                                              scale, live);
    KR_LAUNCHED();
    LossArgs g{};
    g.x = xh;
    g.ldx = ldx;
    g.ldw = ldw;
    g.targets = targets;
    g.lse = lse;
    g.dloss = dloss;
    g.scale = scale;
    g.G = reinterpret_cast<kr_half*>(base + p.G);
    g.G_low = parts == 2 ? g.G + (size_t)p.rows * p.piece : nullptr;
    g.left = reinterpret_cast<float*>(base + p.left);
    g.ldg = p.piece;
    g.N = N;
    g.C = C;
    g.v_all = V;
    g.rows = p.rows;
    ProdArgs d{};
    d.G = g.G;
    d.ldg = g.ldg;
    d.parts = parts;
    d.x = live;
    d.W_all = g.W = reinterpret_cast<const kr_half*>(W);
    d.targets = targets;
    d.left = g.left;
    d.v_all = V;
    d.ldw = ldw;
    d.scale = scale;
    d.dx_part = reinterpret_cast<float*>(base + p.dx_part);
    d.dw_part = reinterpret_cast<float*>(base + p.dw_part);
    d.f32 = out_f32 != 0;
    d.rows = p.rows;
    d.C = C;
    d.dx_splits = p.dx_splits;
    d.dw_splits = p.dw_splits;
    d.N = N;
    d.dx = dx;
    d.dx_direct = p.dx_direct;
    d.dw_run = p.dw_run;
    const int tile = p.big_products ? 256 : 128, gx = (C + tile - 1) / tile;
    for (int i = 0; i < p.pieces; i++) {
        const int v0 = i * p.piece, nv = std::min(V - v0, p.piece);
        g.W = d.W = reinterpret_cast<const kr_half*>(W) + (size_t)v0 * ldw;
        g.V = d.V = nv;
        g.v0 = d.v0 = v0;
        const int rc = logits<true>(g, p.big, s);
        if (rc != KR_OK) return rc;
        d.first = i == 0;
        d.dW = dW ? static_cast<char*>(dW) + (size_t)v0 * C * (out_f32 ? 4 : 2) : nullptr;
        d.dw_items = dW ? (nv + tile - 1) / tile * ((gx + p.dw_run - 1) / p.dw_run) * p.dw_splits : 0;
        d.dx_items = dx ? (p.rows + tile - 1) / tile * gx * p.dx_splits : 0;
        if (p.big_products) grad_products_kernel<4, 2, 8><<<d.dw_items + d.dx_items, 512, 0, s>>>(d);
        else grad_products_kernel<2, 2, 4><<<d.dw_items + d.dx_items, 256, 0, s>>>(d);
        KR_LAUNCHED();
        if (dW && p.dw_splits > 1) {
            const long long n = (long long)nv * C;
            grad_sum_kernel<<<(unsigned)((n / 4 + 255) / 256), 256, 0, s>>>(d.dw_part, n, p.dw_splits, n, scale, out_f32, d.dW,
                                                                           nullptr, 0, 0, nullptr, nullptr, C);
            KR_LAUNCHED();
        }
    }
    if (dx && !p.dx_direct) {
        const long long n = (long long)N * C;
        grad_sum_kernel<<<(unsigned)((n / 4 + 255) / 256), 256, 0, s>>>(d.dx_part, (long long)p.rows * C, p.dx_splits, n,
                                                                       scale, out_f32, dx, d.W_all, ldw, V, targets,
                                                                       d.left, C);
        KR_LAUNCHED();
    }
    return KR_OK;
}

}  // extern "C"
