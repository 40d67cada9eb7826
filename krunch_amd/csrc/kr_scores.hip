// Scores of tokens from rows of logits: the log probability of a given token,
// the row's entropy and its most likely tokens, in one pass over the logits.
//
//   m = max x;  s = sum e^(x - m);  t = sum e^(x - m) (x - m)
//   ln p(i) = (x_i - m) - ln s;     H = ln s - t / s
//
// A row is held in registers (fp16 as it comes, two to a register), so the
// maximum is known before the sums start and memory is read once; rows longer
// than 64 elements a thread of 1024 (32 in fp32) are taken in segments, whose
// (m, s, t) are joined. Sums are fp32, in an order given by the element's index
// alone, so a row's results do not depend on N or on where the row lies.
// Exponentials are 2^(x log2 e - m log2 e): one fused multiply-add and the
// hardware's exp2, the rounding of m log2 e taken back in the sums.
//
// Top tokens: T, the n_top-th largest of 64 disjoint groups' maxima, has at
// least n_top elements >= T and few more where the logits are spread over the
// groups (group = lane: 8 neighbouring tokens, then every 512th). Those go
// to a list in LDS, and each of them counts how many are before it (larger, or
// equal with a lower index): that is its rank. A row with more candidates than
// the list holds (long ties) takes its n_top largest one by one instead.
#include "kr_common.h"
#include "kr_wave.h"
#include "krunch_hip.h"

namespace {

constexpr float kLog2e = 0x1.715476p+0f;
constexpr float kLn2 = 0x1.62e43p-1f;
constexpr int kMaxTop = 64;
constexpr int kListRoom = 512;      // candidates held beside the running top tokens

typedef kr_half8 kr_half8_any __attribute__((aligned(2)));     // rows start at any element
typedef kr_float4 kr_float4_any __attribute__((aligned(4)));

template <typename T> struct Chunk;
template <> struct Chunk<kr_half> {
    static constexpr int n = 8;
    typedef kr_half8 vec;
    typedef kr_half8_any any;
};
template <> struct Chunk<float> {
    static constexpr int n = 4;
    typedef kr_float4 vec;
    typedef kr_float4_any any;
};

struct ScoreArgs {
    const void* logits;
    long long ld;
    int N, V;
    const int32_t* tokens;
    float* logprob;
    float* entropy;
    int n_top;
    float* top_logprob;
    int32_t* top_token;
};

// Orders by value (-0 = +0), then lower index first.
__device__ __forceinline__ uint64_t order_key(float x, uint32_t i) {
    const uint32_t u = __float_as_uint(x + 0.0f);
    const uint32_t o = u & 0x80000000u ? ~u : u | 0x80000000u;
    return (uint64_t)o << 32 | (0xFFFFFFFFu - i);
}
__device__ __forceinline__ float key_value(uint64_t k) {
    const uint32_t o = (uint32_t)(k >> 32);
    return __uint_as_float(o & 0x80000000u ? o & 0x7FFFFFFFu : ~o);
}
__device__ __forceinline__ uint32_t key_index(uint64_t k) { return 0xFFFFFFFFu - (uint32_t)k; }

__device__ __forceinline__ uint64_t wave_max_key(uint64_t k) {
    #pragma unroll
    for (int o = 32; o >= 1; o >>= 1) {
        const uint64_t other = __shfl_xor(k, o);
        k = other > k ? other : k;
    }
    return k;
}

template <int SIZE, int O>
__device__ __forceinline__ float sort_step(float v, int lane) {
    const float w = kr_xor<O>(v);
    const bool larger = ((lane & O) == 0) == (SIZE == 64 || (lane & SIZE) == 0);
    return larger ? fmaxf(v, w) : fminf(v, w);
}
// The 64 lanes' values in descending order.
__device__ __forceinline__ float wave_sort_down(float v, int lane) {
    v = sort_step<2, 1>(v, lane);
    v = sort_step<4, 2>(v, lane); v = sort_step<4, 1>(v, lane);
    v = sort_step<8, 4>(v, lane); v = sort_step<8, 2>(v, lane); v = sort_step<8, 1>(v, lane);
    v = sort_step<16, 8>(v, lane); v = sort_step<16, 4>(v, lane); v = sort_step<16, 2>(v, lane);
    v = sort_step<16, 1>(v, lane);
    v = sort_step<32, 16>(v, lane); v = sort_step<32, 8>(v, lane); v = sort_step<32, 4>(v, lane);
    v = sort_step<32, 2>(v, lane); v = sort_step<32, 1>(v, lane);
    v = sort_step<64, 32>(v, lane); v = sort_step<64, 16>(v, lane); v = sort_step<64, 8>(v, lane);
    v = sort_step<64, 4>(v, lane); v = sort_step<64, 2>(v, lane); v = sort_step<64, 1>(v, lane);
    return v;
}

// What the threads of one row share. W waves work on a row.
template <int W, bool TOP>
struct RowShared {
    float lane_max[W > 1 ? W : 1][64];
    float sum[W], tsum[W];
    float threshold;
    int count;
    uint64_t list[TOP ? kListRoom + kMaxTop : 1];
    uint64_t top[TOP ? kMaxTop : 1];
    uint64_t best[W];
};

// A barrier of the row's threads: the workgroup's, or the wave's own order.
template <int W>
__device__ __forceinline__ void row_sync() {
    if constexpr (W > 1) __syncthreads();
    else {
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }
}

// W waves per row, U chunks of 16 bytes per thread, 4 / W rows (at least one)
// per workgroup.
template <typename T, int W, int U, bool TOP>
__global__ void __launch_bounds__(W >= 4 ? 64 * W : 256, W == 16 ? (sizeof(T) == 2 ? 8 : 4) : 6)
scores_kernel(ScoreArgs g) {
    constexpr int kRows = W >= 4 ? 1 : 4 / W;
    constexpr int CH = Chunk<T>::n, TH = 64 * W, kSegment = TH * CH * U;
    typedef typename Chunk<T>::vec vec;
    __shared__ RowShared<W, TOP> shared_rows[kRows];
    const int lane = threadIdx.x & 63;
    const int wave = W > 1 ? threadIdx.x / 64 % W : 0;
    const int tid = 64 * wave + lane;
    const int slot = kRows > 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x / TH) : 0;
    RowShared<W, TOP>& sh = shared_rows[slot];
    const long long row = (long long)blockIdx.x * kRows + slot;
    if (kRows > 1 && row >= g.N) return;    // a whole wave: rows of W = 1 share nothing
    const T* x0 = reinterpret_cast<const T*>(g.logits) + row * g.ld;
    const int token = g.tokens[row];
    const bool named = token >= 0 && token < g.V;
    const float x_token = named ? (float)x0[token] : 0.0f;

    float M = -INFINITY, S = 0.0f, Q = 0.0f;   // running maximum, sums of e and e * (x - M) log2 e
    int kept = 0;                               // entries of sh.top
    for (int base = 0; base < g.V; base += kSegment) {
        const T* xs = x0 + base;
        const int n = g.V - base < kSegment ? g.V - base : kSegment;
        vec x[U];
        #pragma unroll
        for (int u = 0; u < U; u++) {
            const int i = (u * TH + tid) * CH;
            #pragma unroll
            for (int e = 0; e < CH; e++) x[u][e] = (T)-INFINITY;
            if (i + CH <= n) {
                x[u] = *reinterpret_cast<const typename Chunk<T>::any*>(xs + i);
            } else if (i < n) {
                #pragma unroll
                for (int e = 0; e < CH; e++)
                    if (i + e < n) x[u][e] = xs[i + e];
            }
        }
        T chunk_max[U];
        float mine = -INFINITY;
        #pragma unroll
        for (int u = 0; u < U; u++) {
            vec v = x[u];
            if constexpr (CH == 8) {
                kr_half4 h = __builtin_elementwise_max(
                    __builtin_shufflevector(v, v, 0, 1, 2, 3), __builtin_shufflevector(v, v, 4, 5, 6, 7));
                typedef kr_half half2v __attribute__((ext_vector_type(2)));
                half2v p = __builtin_elementwise_max(__builtin_shufflevector(h, h, 0, 1),
                                                     __builtin_shufflevector(h, h, 2, 3));
                chunk_max[u] = __builtin_elementwise_max(p[0], p[1]);
            } else {
                chunk_max[u] = (T)fmaxf(fmaxf((float)v[0], (float)v[1]), fmaxf((float)v[2], (float)v[3]));
            }
            mine = fmaxf(mine, (float)chunk_max[u]);
        }
        // maximum per lane over the row's waves (the groups of T), then of all
        float group = mine;
        if constexpr (W > 1) {
            sh.lane_max[wave][lane] = mine;
            row_sync<W>();
            #pragma unroll
            for (int w = 0; w < W; w++) group = fmaxf(group, sh.lane_max[w][lane]);
        }
        float m = kr_wave_reduce(group, [](float a, float b) { return fmaxf(a, b); });
        if (TOP && wave == 0) {
            const float sorted = wave_sort_down(group, lane);
            const float th = __int_as_float(
                __builtin_amdgcn_readlane(__float_as_int(sorted), g.n_top - 1));
            if (lane == 0) {
                sh.threshold = th;
                sh.count = 0;
            }
        }
        if (m == -INFINITY) m = 0.0f;           // nothing above -inf: every e is 0 (or NaN)
        float s = 0.0f, q = 0.0f;
        const float ml = m * kLog2e;
        #pragma unroll
        for (int u = 0; u < U; u++) {
            if ((u * TH + 64 * wave) * CH >= n) break;     // wave-uniform: nothing of the row here
            #pragma unroll
            for (int e = 0; e < CH; e++) {
                float a;
                if constexpr (CH == 8) a = __builtin_fmaf((float)x[u][e], kLog2e, -ml);
                else a = ((float)x[u][e] - m) * kLog2e;
                const float ex = __builtin_amdgcn_exp2f(a);
                s += ex;
                q = __builtin_fmaf(ex, fmaxf(a, -1000.0f), q);   // e^-inf * -inf = 0
            }
        }
        s = kr_wave_reduce(s, [](float a, float b) { return a + b; });
        q = kr_wave_reduce(q, [](float a, float b) { return a + b; });
        if constexpr (W > 1) {
            if (lane == 0) {
                sh.sum[wave] = s;
                sh.tsum[wave] = q;
            }
            row_sync<W>();
            s = 0.0f;
            q = 0.0f;
            #pragma unroll
            for (int w = 0; w < W; w++) {
                s += sh.sum[w];
                q += sh.tsum[w];
            }
        } else {
            row_sync<W>();
        }
        if constexpr (CH == 8) {
            // every e is 2^b too large, b the rounding of ml
            const float b = __builtin_fmaf(m, kLog2e, -ml), f = __builtin_amdgcn_exp2f(-b);
            q = f * __builtin_fmaf(-b, s, q);
            s = f * s;
        }
        if (base == 0) {
            M = m;
            S = s;
            Q = q;
        } else if (s != 0.0f) {                 // (NaN too)
            // join: both sides relative to the larger maximum; an empty side adds nothing
            if (S == 0.0f) {
                M = m;
                S = s;
                Q = q;
            } else {
                const float top = fmaxf(M, m);
                const float d0 = fmaxf((M - top) * kLog2e, -1000.0f);
                const float d1 = fmaxf((m - top) * kLog2e, -1000.0f);
                const float f0 = __builtin_amdgcn_exp2f(d0), f1 = __builtin_amdgcn_exp2f(d1);
                Q = f0 * __builtin_fmaf(d0, S, Q) + f1 * __builtin_fmaf(d1, s, q);
                S = f0 * S + f1 * s;
                M = top;
            }
        }
        if constexpr (TOP) {
            // chunks with a candidate, few: read again, so that no element stays
            // converted, with its key, from the sums on (146 spilled registers)
            const float th = sh.threshold;
            uint32_t hit = 0;
            #pragma unroll
            for (int u = 0; u < U; u++)
                hit |= ((float)chunk_max[u] >= th && (float)chunk_max[u] > -INFINITY) ? 1u << u : 0u;
            while (hit) {
                const int i = ((__ffs(hit) - 1) * TH + tid) * CH;
                hit &= hit - 1;
                #pragma unroll 1
                for (int e = 0; e < CH && i + e < n; e++) {
                    const float xe = (float)xs[i + e];
                    if (xe >= th && xe > -INFINITY) {
                        const int at = atomicAdd(&sh.count, 1);
                        if (at < kListRoom) sh.list[at] = order_key(xe, (uint32_t)(base + i + e));
                    }
                }
            }
            row_sync<W>();
            const int found = sh.count;
            if (found <= kListRoom) {
                // rank among the candidates and the earlier segments' top tokens
                if (tid < kept) sh.list[found + tid] = sh.top[tid];
                row_sync<W>();
                const int all = found + kept;
                for (int c = tid; c < all; c += TH) {
                    const uint64_t k = sh.list[c];
                    int rank = 0;
                    for (int j = 0; j < all; j++) rank += sh.list[j] > k;
                    if (rank < g.n_top) sh.top[rank] = k;
                }
                kept = all < g.n_top ? all : g.n_top;
            } else {
                // one after the other, each the largest below the one before
                if (tid < kept) sh.list[tid] = sh.top[tid];
                row_sync<W>();
                const int had = kept;
                uint64_t last = ~0ull;
                for (kept = 0; kept < g.n_top; kept++) {
                    uint64_t k = 0;
                    #pragma unroll 1
                    for (int i = tid; i < n; i += TH) {
                        const float xe = (float)xs[i];
                        const uint64_t c = order_key(xe, (uint32_t)(base + i));
                        if (xe > -INFINITY && c < last && c > k) k = c;
                    }
                    if (tid < had && sh.list[tid] < last && sh.list[tid] > k) k = sh.list[tid];
                    k = wave_max_key(k);
                    if constexpr (W > 1) {
                        if (lane == 0) sh.best[wave] = k;
                        row_sync<W>();
                        for (int w = 0; w < W; w++) k = sh.best[w] > k ? sh.best[w] : k;
                        row_sync<W>();
                    }
                    if (k == 0) break;          // the row has no more
                    if (tid == 0) sh.top[kept] = k;
                    last = k;
                }
            }
            row_sync<W>();
        }
    }

    // S: 0 = nothing above -inf, NaN = a NaN or +inf in the row
    const float ln_s = __logf(S);
    if (tid == 0) {
        float lp = (x_token - M) - ln_s;
        float h = ln_s - kLn2 * (Q / S);
        if (S == 0.0f) {
            lp = -INFINITY;
            h = 0.0f;
        }
        if (token == -1) lp = 0.0f;
        else if (!named) lp = NAN;
        g.logprob[row] = lp;
        g.entropy[row] = h;
    }
    if (TOP && tid < g.n_top) {
        const bool good = S == S, there = good && tid < kept;
        const uint64_t k = there ? sh.top[tid] : 0;
        const size_t o = (size_t)row * g.n_top + tid;
        g.top_logprob[o] = there ? (key_value(k) - M) - ln_s : good ? -INFINITY : NAN;
        g.top_token[o] = there ? (int32_t)key_index(k) : -1;
    }
}

template <typename T, int W, int U>
void launch(const ScoreArgs& g, hipStream_t s) {
    constexpr int rows = W >= 4 ? 1 : 4 / W;
    const int threads = W >= 4 ? 64 * W : 256;
    const int grid = (g.N - 1) / rows + 1;
    if (g.n_top) scores_kernel<T, W, U, true><<<grid, threads, 0, s>>>(g);
    else scores_kernel<T, W, U, false><<<grid, threads, 0, s>>>(g);
}

template <typename T>
void launch_by_width(const ScoreArgs& g, hipStream_t s) {
    constexpr int CH = Chunk<T>::n;
    if (g.V <= 64 * CH) launch<T, 1, 1>(g, s);
    else if (g.V <= 256 * CH) launch<T, 1, 4>(g, s);
    else if (g.V <= 4 * 256 * CH) launch<T, 4, 4>(g, s);
    else launch<T, 16, 8>(g, s);
}

}  // namespace

extern "C" int kr_token_scores(const void* logits, int logits_f32, int N, int V, long long ld,
                               const int32_t* tokens, float* logprob, float* entropy, int n_top,
                               float* top_logprob, int32_t* top_token, void* stream) {
    KR_REQUIRE(N >= 0, "kr_token_scores: N=%d", N);
    KR_REQUIRE(V >= 1 && ld >= V, "kr_token_scores: V=%d, ld=%lld", V, ld);
    KR_REQUIRE(n_top >= 0 && n_top <= kMaxTop && n_top <= V,
               "kr_token_scores: n_top=%d must be in 0..%d and at most V=%d", n_top, kMaxTop, V);
    if (N == 0) return KR_OK;
    KR_REQUIRE(logits && tokens && logprob && entropy, "kr_token_scores: null pointer");
    KR_REQUIRE(n_top == 0 || (top_logprob && top_token), "kr_token_scores: null top pointer");
    KR_REQUIRE(((uintptr_t)logits & (logits_f32 ? 3 : 1)) == 0, "kr_token_scores: misaligned logits");
    const ScoreArgs g{logits, ld, N, V, tokens, logprob, entropy, n_top, top_logprob, top_token};
    if (logits_f32) launch_by_width<float>(g, kr_stream(stream));
    else launch_by_width<kr_half>(g, kr_stream(stream));
    KR_LAUNCHED();
    return KR_OK;
}
