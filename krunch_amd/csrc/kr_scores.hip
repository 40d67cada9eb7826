// Scores of tokens from rows of logits: the log probability of a given token,
// the row's entropy and its most likely tokens, in one pass over the logits.
//
//   m = max x;  s = sum e^(x - m);  t = sum e^(x - m) (x - m)
//   ln p(i) = (x_i - m) - ln s;     H = ln s - t / s
//
// One pass over memory: a thread keeps a running maximum and the two sums relative
// to it, rescaled where a block of its chunks has a larger one; the threads' are
// joined at the row's end. Sums are fp32, in an order given by the element's index
// alone, so a row's results do not depend on N or on where the row lies. A block of
// at most 32 terms is summed by itself, and a thread's blocks with their rounding
// errors carried along, so the error does not grow with V: in one chain, equal
// logits of V = 2^24 came out 5e-4 off.
// Exponentials are 2^(x log2 e - m log2 e): for fp16 one fused multiply-add and the
// hardware's exp2, sums being relative to the rounded m log2 e.
//
// Top tokens: T, the n_top-th largest of 16 (n_top <= 8) or 64 disjoint groups'
// maxima, has at least n_top elements >= T and few more where the logits are
// spread over the groups (64: lanes, so 8 neighbouring tokens, then every 512th).
// Threads with a maximum >= T, few, are listed and their chunks read again (from
// the L2; a row of one wave has them in registers), and each element >= T counts
// how many are before it (larger, or equal with a lower index): that is its rank. A
// row with more of them than there is room for (long ties) takes its n_top largest
// one by one instead.
#include "kr_common.h"
#include "kr_wave.h"
#include "krunch_hip.h"

#include <type_traits>

namespace {

constexpr float kLog2e = 0x1.715476p+0f;
constexpr float kLn2 = 0x1.62e43p-1f;
constexpr int kMaxTop = 32;

template <typename T> struct Chunk;
template <> struct Chunk<kr_half> {
    static constexpr int n = 8;
    typedef kr_half8 vec;
};
template <> struct Chunk<float> {
    static constexpr int n = 4;
    typedef kr_float4 vec;
};

// 16 bytes of a row: rows, and the last chunk of a row, start at any element.
typedef kr_int4 int4_any __attribute__((aligned(2)));
static_assert(alignof(int4_any) <= alignof(kr_half), "chunks start at any element");

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

// One step of a bitonic sort. LAST: of the last merge, all descending.
template <int SIZE, int O, bool LAST = SIZE == 64>
__device__ __forceinline__ float sort_step(float v, int lane) {
    const float w = kr_xor<O>(v);
    const bool larger = ((lane & O) == 0) == (LAST || (lane & SIZE) == 0);
    return larger ? fmaxf(v, w) : fminf(v, w);
}
template <bool LAST>
__device__ __forceinline__ float sort_16(float v, int lane) {
    v = sort_step<2, 1>(v, lane);
    v = sort_step<4, 2>(v, lane); v = sort_step<4, 1>(v, lane);
    v = sort_step<8, 4>(v, lane); v = sort_step<8, 2>(v, lane); v = sort_step<8, 1>(v, lane);
    v = sort_step<16, 8, LAST>(v, lane); v = sort_step<16, 4, LAST>(v, lane);
    v = sort_step<16, 2, LAST>(v, lane);
    return sort_step<16, 1, LAST>(v, lane);
}
// The k-th largest of the 64 lanes' values, or with k <= 8 of the maxima of the 16
// groups of lanes l, l + 16, l + 32, l + 48: less spread over the row, but half
// the steps, and without exchanges between the wave's quarters.
__device__ __forceinline__ float kth_largest(float v, int lane, int k) {
    if (k <= 8) {
        v = fmaxf(v, kr_xor<16>(v));
        v = fmaxf(v, kr_xor<32>(v));
    }
    v = sort_16<false>(v, lane);
    if (k > 8) {
        v = sort_step<32, 16>(v, lane); v = sort_step<32, 8>(v, lane); v = sort_step<32, 4>(v, lane);
        v = sort_step<32, 2>(v, lane); v = sort_step<32, 1>(v, lane);
        v = sort_step<64, 32>(v, lane); v = sort_step<64, 16>(v, lane); v = sort_step<64, 8>(v, lane);
        v = sort_step<64, 4>(v, lane); v = sort_step<64, 2>(v, lane); v = sort_step<64, 1>(v, lane);
    }
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), k - 1));
}

// What the threads of one row share. W waves work on a row.
template <int W, bool TOP>
struct RowShared {
    static constexpr int kThreads = TOP ? 96 : 1;        // with candidates
    static constexpr int kList = TOP ? 384 : 1;          // candidates
    float lane_max[W > 1 ? W : 1][64];
    float sum[W], tsum[W];
    float threshold;
    int threads, count;
    int thread[kThreads];
    uint64_t list[kList];
    uint64_t top[TOP ? kMaxTop : 1];
    uint64_t best[W];
};

// Element words of a row shorter than a chunk, and -inf past it.
template <typename T>
__device__ __forceinline__ kr_int4 read_short(const T* x, int i, int n) {
    kr_int4 v;
    #pragma unroll
    for (int j = 0; j < 4; j++) {
        if constexpr (sizeof(T) == 4) {
            v[j] = i + j < n ? __float_as_int((float)x[i + j]) : (int)0xFF800000;
        } else {
            const uint16_t* h = reinterpret_cast<const uint16_t*>(x);
            const uint32_t lo = i + 2 * j < n ? h[i + 2 * j] : 0xFC00u;
            const uint32_t hi = i + 2 * j + 1 < n ? h[i + 2 * j + 1] : 0xFC00u;
            v[j] = (int)(lo | hi << 16);
        }
    }
    return v;
}
template <typename T>
__device__ __forceinline__ float chunk_max(kr_int4 raw) {
    const typename Chunk<T>::vec v = __builtin_bit_cast(typename Chunk<T>::vec, raw);
    if constexpr (sizeof(T) == 2) {
        typedef kr_half half2v __attribute__((ext_vector_type(2)));
        const kr_half4 h = __builtin_elementwise_max(__builtin_shufflevector(v, v, 0, 1, 2, 3),
                                                     __builtin_shufflevector(v, v, 4, 5, 6, 7));
        const half2v p = __builtin_elementwise_max(__builtin_shufflevector(h, h, 0, 1),
                                                   __builtin_shufflevector(h, h, 2, 3));
        return (float)__builtin_elementwise_max(p[0], p[1]);
    } else {
        return fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3]));
    }
}
// The first d elements of a chunk become -inf.
template <typename T>
__device__ __forceinline__ kr_int4 without_first(kr_int4 v, int d) {
    #pragma unroll
    for (int j = 0; j < 4; j++) {
        if constexpr (sizeof(T) == 4) {
            if (j < d) v[j] = (int)0xFF800000;
        } else {
            const uint32_t w = (uint32_t)v[j];
            v[j] = (int)(2 * j + 1 < d ? 0xFC00FC00u : 2 * j < d ? (w & 0xFFFF0000u) | 0xFC00u : w);
        }
    }
    return v;
}

// sum + x, and what the addition rounded off to low: exactly where |sum| >= |x|.
// Elsewhere (x has the sum's sign, or the size of a rounding) the sum more than
// doubles, so what those additions lose, half a last place each, comes to one last
// place of the final sum in all. 8 operations a block: 8192 x 50277 143.1 -> 143.5 us.
__device__ __forceinline__ void add_carried(float& sum, float& low, float x) {
    const float t = sum + x;
    low += x - (t - sum);
    sum = t;
}

// A barrier of the row's threads: the workgroup's, or the wave's own order.
template <int W>
__device__ __forceinline__ void row_sync() {
    if constexpr (W > 1) __syncthreads();
    else {
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }
}

// W waves per row, U chunks of 16 bytes per thread at a time; four rows a workgroup
// with W = 1, else one.
// Bound: memory with many rows (8192 x 50277 fp16 143 us, with 8 top 153: 5.8 and 5.4
// TB/s, fp32 270: 6.1; holding rows in registers and sums made anew after the
// maximum 165, one row per 16 waves 194); latency with few: one row of 50277 with 5 top
// 7.7 us, of which 3.6 is any launch's and 2 are T, the list and the ranks.
template <typename T, int W, int U, bool TOP>
__global__ void __launch_bounds__(W > 1 ? 64 * W : 256, 8)
scores_kernel(ScoreArgs g) {
    constexpr int kRows = W > 1 ? 1 : 4;
    constexpr int CH = Chunk<T>::n, TH = 64 * W;
    typedef typename Chunk<T>::vec vec;
    __shared__ RowShared<W, TOP> shared_rows[kRows];
    const int lane = threadIdx.x & 63;
    const int wave = W > 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x / 64 % W) : 0;
    const int tid = 64 * wave + lane;
    const int slot = kRows > 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x / TH) : 0;
    RowShared<W, TOP>& sh = shared_rows[slot];
    const long long row = (long long)blockIdx.x * kRows + slot;
    if (kRows > 1 && row >= g.N) return;    // a whole wave: rows of W = 1 share nothing
    const int V = g.V;
    const T* x = reinterpret_cast<const T*>(g.logits) + row * g.ld;
    const int token = g.tokens[row];
    const bool named = token >= 0 && token < V;
    const float x_token = named ? (float)x[token] : 0.0f;

    // Chunk c of the row starts at element c * CH; one that ends past the row is
    // read from the row's last 16 bytes, without what belongs to the one before.
    auto chunk_start = [&](int c) { return min(c * CH, V - CH); };
    const int chunks = (V + CH - 1) / CH;
    // U chunks of the thread from chunk c0 + lane on, TH apart. fp16 rows that start
    // in the middle of a 4-byte word are read by the words around: reads of 16 bytes
    // run at full speed from any 4-byte boundary, and 26% slower over rows of which
    // half have none (8192 x 50277 held in registers: 165 us, 209). The last element
    // is read by itself: the word that it begins may end behind the row.
    auto read_block = [&](int c0, kr_int4 (&raw)[U], auto odd_row) {
        constexpr bool ODD = decltype(odd_row)::value;
        uint32_t next[U];
        #pragma unroll
        for (int u = 0; u < U; u++) {
            const T* at = x + chunk_start(c0 + u * TH + lane);
            raw[u] = *reinterpret_cast<const int4_any*>(at - (ODD ? 1 : 0));
            if (ODD) next[u] = reinterpret_cast<const uint16_t*>(at)[7];
        }
        if (ODD) {
            #pragma unroll
            for (int u = 0; u < U; u++)
                #pragma unroll
                for (int j = 0; j < 4; j++)
                    raw[u][j] = (int)__builtin_amdgcn_alignbit(
                        j < 3 ? (uint32_t)raw[u][j + 1] : next[u], (uint32_t)raw[u][j], 16);
        }
        if ((c0 + (U - 1) * TH + 64) * CH > V) {
            #pragma unroll
            for (int u = 0; u < U; u++) {
                const int c = c0 + u * TH + lane;
                raw[u] = without_first<T>(raw[u], c * CH - chunk_start(c));
            }
        }
    };
    const std::integral_constant<bool, true> odd;
    const std::integral_constant<bool, false> even;
    const bool is_odd = sizeof(T) == 2 && ((uintptr_t)x & 2);
    // m: maximum; ref: what the sums s of e and q of e a are relative to, in log2
    // (fp32: the maximum itself, whose log2 e multiple may overflow)
    float m = -INFINITY, ref = 0.0f, s = 0.0f, q = 0.0f;
    auto reference = [](float top) { return top == -INFINITY ? 0.0f : CH == 8 ? top * kLog2e : top; };
    float s_low = 0.0f, q_low = 0.0f;     // what the additions of blocks rounded off
    auto add = [&](const kr_int4 (&raw)[U]) {
        float sb = 0.0f, qb = 0.0f;
        #pragma unroll
        for (int u = 0; u < U; u++) {
            const vec v = __builtin_bit_cast(vec, raw[u]);
            #pragma unroll
            for (int e = 0; e < CH; e++) {
                float a;
                if constexpr (CH == 8) a = __builtin_fmaf((float)v[e], kLog2e, -ref);
                else a = ((float)v[e] - ref) * kLog2e;
                const float ex = __builtin_amdgcn_exp2f(a);
                sb += ex;
                qb = __builtin_fmaf(ex, fmaxf(a, -1000.0f), qb);   // e^-inf * -inf = 0
            }
        }
        if constexpr (W == 1) {
            s = sb;
            q = qb;
        } else {
            add_carried(s, s_low, sb);
            add_carried(q, q_low, qb);
        }
    };
    // s and q relative to `to`, which is not below ref; with m = -inf, nothing is
    // in them but, perhaps, NaN
    auto rescale = [&](float to) {
        if (m != -INFINITY) {
            const float d = fmaxf(CH == 8 ? ref - to : (ref - to) * kLog2e, -1000.0f);
            const float f = __builtin_amdgcn_exp2f(d);
            q = f * __builtin_fmaf(d, s, q);
            s = f * s;
            q_low = f * __builtin_fmaf(d, s_low, q_low);
            s_low = f * s_low;
        }
        ref = to;
    };
    kr_int4 raw[U];
    if constexpr (W == 1) {
        // the whole row is one block of its wave
        if (is_odd) read_block(0, raw, odd);
        else read_block(0, raw, even);
        #pragma unroll
        for (int u = 0; u < U; u++) m = fmaxf(m, chunk_max<T>(raw[u]));
    } else {
        auto walk = [&](auto odd_row) {
            for (int c0 = 64 * wave; c0 < chunks; c0 += U * TH) {
                read_block(c0, raw, odd_row);
                float top = -INFINITY;
                #pragma unroll
                for (int u = 0; u < U; u++) top = fmaxf(top, chunk_max<T>(raw[u]));
                if (__any(top > m)) {
                    top = fmaxf(top, m);
                    rescale(reference(top));
                    m = top;
                }
                add(raw);
            }
        };
        if (is_odd) walk(odd);
        else walk(even);
    }

    // maximum per lane over the row's waves (the groups of T), then of all
    float group = m;
    if constexpr (W > 1) {
        sh.lane_max[wave][lane] = m;
        row_sync<W>();
        #pragma unroll
        for (int w = 0; w < W; w++) group = fmaxf(group, sh.lane_max[w][lane]);
    }
    const float M = kr_wave_reduce(group, [](float a, float b) { return fmaxf(a, b); });
    if constexpr (W == 1) {
        ref = reference(M);
        add(raw);
    } else {
        rescale(reference(M));
        s += s_low;
        q += q_low;
    }
    s = kr_wave_reduce(s, [](float a, float b) { return a + b; });
    q = kr_wave_reduce(q, [](float a, float b) { return a + b; });
    if (TOP && wave == W - 1) {
        const float th = kth_largest(group, lane, g.n_top);
        if (lane == 0) {
            sh.threshold = th;
            sh.threads = 0;
            sh.count = 0;
        }
    }
    if constexpr (W > 1) {
        if (lane == 0) {
            sh.sum[wave] = s;
            sh.tsum[wave] = q;
        }
    }
    row_sync<W>();
    int kept = 0;
    if constexpr (TOP) {
        const float th = sh.threshold;
        int all = 0;
        bool room = true;
        if constexpr (W == 1) {
            #pragma unroll
            for (int u = 0; u < U; u++) {
                if (!__any(chunk_max<T>(raw[u]) >= th)) continue;
                const vec v = __builtin_bit_cast(vec, raw[u]);
                const int start = chunk_start(u * TH + lane);
                #pragma unroll
                for (int e = 0; e < CH; e++) {
                    const float xe = (float)v[e];
                    const bool in = xe >= th && xe > -INFINITY;
                    const uint64_t mask = __ballot(in);
                    const int at = all + __popcll(mask & ((1ull << lane) - 1));
                    if (in && at < sh.kList) sh.list[at] = order_key(xe, (uint32_t)(start + e));
                    all += __popcll(mask);
                }
            }
            row_sync<W>();
            room = all <= sh.kList;
        } else {
            if (m >= th && m > -INFINITY) {
                const int at = atomicAdd(&sh.threads, 1);
                if (at < sh.kThreads) sh.thread[at] = tid;
            }
            row_sync<W>();
            const int threads = sh.threads;
            if (threads <= sh.kThreads) {
                const int per = (chunks + TH - 1) / TH;       // chunks of a thread
                for (int i = tid; i < threads * per; i += TH) {
                    const int c = sh.thread[i / per] + i % per * TH;
                    if (c >= chunks) continue;
                    const int start = chunk_start(c);
                    vec v;
                    __builtin_memcpy(&v, x + start, 16);
                    #pragma unroll
                    for (int e = 0; e < CH; e++) {
                        const float xe = (float)v[e];
                        if (xe >= th && xe > -INFINITY && start + e >= c * CH) {
                            const int at = atomicAdd(&sh.count, 1);
                            if (at < sh.kList) sh.list[at] = order_key(xe, (uint32_t)(start + e));
                        }
                    }
                }
            }
            row_sync<W>();
            all = sh.count;
            room = threads <= sh.kThreads && all <= sh.kList;
        }
        if (room) {
            if (wave > 0) return;
            for (int c = lane; c < all; c += 64) {
                const uint64_t k = sh.list[c];
                int rank = 0;
                #pragma unroll 4
                for (int j = 0; j < all; j++) rank += sh.list[j] > k;
                if (rank < g.n_top) sh.top[rank] = k;
            }
            kept = all < g.n_top ? all : g.n_top;
            row_sync<1>();
        } else {
            // one after the other, each the largest below the one before
            uint64_t last = ~0ull;
            for (; kept < g.n_top; kept++) {
                uint64_t k = 0;
                #pragma unroll 1
                for (int i = tid; i < V; i += TH) {
                    const float v = (float)x[i];
                    const uint64_t c = order_key(v, (uint32_t)i);
                    if (v > -INFINITY && c < last && c > k) k = c;
                }
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
            row_sync<W>();
        }
    }
    if (wave > 0) return;

    if constexpr (W > 1) {
        s = 0.0f;
        q = 0.0f;
        #pragma unroll
        for (int w = 0; w < W; w++) {
            s += sh.sum[w];
            q += sh.tsum[w];
        }
    }
    // s: 0 = nothing above -inf, NaN = a NaN or +inf in the row. With M log2 e
    // rounded by b, every e is 2^b too large
    const float base = M == -INFINITY ? 0.0f : M;
    const float b = CH == 8 ? __builtin_fmaf(base, kLog2e, -ref) : 0.0f;
    const float ln_s = __logf(s) - b * kLn2;
    if (lane == 0) {
        float lp = (x_token - base) - ln_s;
        float h = __logf(s) - kLn2 * (q / s);
        lp = lp > 0.0f ? 0.0f : lp;           // a rounding of a token of probability 1
        h = h < 0.0f ? 0.0f : h;
        if (s == 0.0f) {
            lp = -INFINITY;
            h = 0.0f;
        }
        if (token == -1) lp = 0.0f;
        else if (!named) lp = NAN;
        g.logprob[row] = lp;
        g.entropy[row] = h;
    }
    if (TOP && lane < g.n_top) {
        const bool good = s == s, there = good && lane < kept;
        const uint64_t k = there ? sh.top[lane] : 0;
        const size_t o = (size_t)row * g.n_top + lane;
        const float lp = (key_value(k) - base) - ln_s;
        g.top_logprob[o] = there ? (lp > 0.0f ? 0.0f : lp) : good ? -INFINITY : NAN;
        g.top_token[o] = there ? (int32_t)key_index(k) : -1;
    }
}

// Short rows: 16 lanes have a row, so a wave's reductions and sort serve four. U
// chunks of 16 bytes per lane, in registers; n_top <= 8, T the n_top-th largest of
// the 16 lanes' maxima. Rows of one wave may start at different halves of a word, so
// fp16 is always read as four words and the last element, shifted by 0 or 16 bits.
// Bound: memory without top tokens (100000 x 512 fp32 36.6 us, 5.6 TB/s), issue with
// them (3 top of 256 fp16: 12.6 us without, 22.5); 16 rows a workgroup.
constexpr int kShortChunks = 24, kShortList = 64;      // with candidates, and candidates, of a row

template <typename T, int U, bool TOP>
__global__ void __launch_bounds__(256, 8) scores_short_kernel(ScoreArgs g) {
    constexpr int CH = Chunk<T>::n;
    typedef typename Chunk<T>::vec vec;
    __shared__ kr_int4 hit_chunk[TOP ? 16 : 1][kShortChunks];
    __shared__ int hit_at[TOP ? 16 : 1][kShortChunks];
    __shared__ int hits[16], found[16];
    __shared__ uint64_t list[TOP ? 16 : 1][kShortList];
    __shared__ uint64_t best[TOP ? 16 : 1][8];
    const int lane = threadIdx.x & 63, l = lane & 15, slot = threadIdx.x >> 4;
    const long long row = (long long)blockIdx.x * 16 + slot;
    const bool there = row < g.N;
    const long long r = there ? row : g.N - 1;      // past N: the last row, not written
    const int V = g.V;
    const T* x = reinterpret_cast<const T*>(g.logits) + r * g.ld;
    const int token = g.tokens[r];
    const bool named = token >= 0 && token < V;
    const float x_token = named ? (float)x[token] : 0.0f;
    if (TOP && l == 0) hits[slot] = found[slot] = 0;
    auto chunk_start = [&](int u) { return V < CH ? l * CH : min((u * 16 + l) * CH, V - CH); };
    kr_int4 raw[U];
    float m = -INFINITY;
    if (V < CH) {
        #pragma unroll
        for (int u = 0; u < U; u++) raw[u] = read_short(x, (u * 16 + l) * CH, V);
    } else {
        const int odd = sizeof(T) == 2 ? (int)((uintptr_t)x >> 1 & 1) : 0;
        uint32_t next[U];
        #pragma unroll
        for (int u = 0; u < U; u++) {
            const T* at = x + chunk_start(u);
            raw[u] = *reinterpret_cast<const int4_any*>(at - odd);
            if (sizeof(T) == 2) next[u] = reinterpret_cast<const uint16_t*>(at)[7];
        }
        #pragma unroll
        for (int u = 0; u < U; u++) {
            if (sizeof(T) == 2) {
                #pragma unroll
                for (int j = 0; j < 4; j++)
                    raw[u][j] = (int)__builtin_amdgcn_alignbit(
                        j < 3 ? (uint32_t)raw[u][j + 1] : next[u], (uint32_t)raw[u][j], 16 * odd);
            }
            if ((u + 1) * 16 * CH > V) raw[u] = without_first<T>(raw[u], (u * 16 + l) * CH - chunk_start(u));
        }
    }
    #pragma unroll
    for (int u = 0; u < U; u++) m = fmaxf(m, chunk_max<T>(raw[u]));
    float M = m;
    M = fmaxf(M, kr_xor<8>(M));
    M = fmaxf(M, kr_xor<4>(M));
    M = fmaxf(M, kr_xor<2>(M));
    M = fmaxf(M, kr_xor<1>(M));
    const float base = M == -INFINITY ? 0.0f : M;
    const float ref = CH == 8 ? base * kLog2e : base;
    float s = 0.0f, q = 0.0f;
    #pragma unroll
    for (int u = 0; u < U; u++) {
        const vec v = __builtin_bit_cast(vec, raw[u]);
        #pragma unroll
        for (int e = 0; e < CH; e++) {
            const float a = CH == 8 ? __builtin_fmaf((float)v[e], kLog2e, -ref) : ((float)v[e] - ref) * kLog2e;
            const float ex = __builtin_amdgcn_exp2f(a);
            s += ex;
            q = __builtin_fmaf(ex, fmaxf(a, -1000.0f), q);
        }
    }
    s += kr_xor<8>(s);
    s += kr_xor<4>(s);
    s += kr_xor<2>(s);
    s += kr_xor<1>(s);
    q += kr_xor<8>(q);
    q += kr_xor<4>(q);
    q += kr_xor<2>(q);
    q += kr_xor<1>(q);
    const float b = CH == 8 ? __builtin_fmaf(base, kLog2e, -ref) : 0.0f;
    const float log_s = __logf(s), ln_s = log_s - b * kLn2;
    if (there && l == 0) {
        float lp = (x_token - base) - ln_s;
        float h = log_s - kLn2 * (q / s);
        lp = lp > 0.0f ? 0.0f : lp;           // a rounding of a token of probability 1
        h = h < 0.0f ? 0.0f : h;
        if (s == 0.0f) {
            lp = -INFINITY;
            h = 0.0f;
        }
        if (token == -1) lp = 0.0f;
        else if (!named) lp = NAN;
        g.logprob[row] = lp;
        g.entropy[row] = h;
    }
    if constexpr (TOP) {
        const float th = __shfl(sort_16<true>(m, lane), (lane & 48) + g.n_top - 1);
        row_sync<1>();
        #pragma unroll
        for (int u = 0; u < U; u++) {
            const float c = chunk_max<T>(raw[u]);
            if (c >= th && c > -INFINITY) {
                const int at = atomicAdd(&hits[slot], 1);
                if (at < kShortChunks) {
                    hit_chunk[slot][at] = raw[u];
                    hit_at[slot][at] = chunk_start(u);
                }
            }
        }
        row_sync<1>();
        const int chunks = hits[slot];
        if (chunks <= kShortChunks) {
            for (int i = l; i < chunks * CH; i += 16) {
                const float v = (float)reinterpret_cast<const T*>(hit_chunk[slot])[i];
                if (v >= th && v > -INFINITY) {
                    const int at = atomicAdd(&found[slot], 1);
                    if (at < kShortList)
                        list[slot][at] = order_key(v, (uint32_t)(hit_at[slot][i / CH] + i % CH));
                }
            }
            if (l < 8) best[slot][l] = 0;
        }
        row_sync<1>();
        const int all = found[slot];
        if (chunks <= kShortChunks && all <= kShortList) {
            for (int i = l; i < all; i += 16) {
                const uint64_t k = list[slot][i];
                int rank = 0;
                #pragma unroll 4
                for (int j = 0; j < all; j++) rank += list[slot][j] > k;
                if (rank < g.n_top) best[slot][rank] = k;
            }
            row_sync<1>();
        } else {
            // one after the other, each the largest below the one before
            uint64_t last = ~0ull;
            for (int kept = 0; kept < g.n_top; kept++) {
                uint64_t k = 0;
                #pragma unroll 1
                for (int i = l; i < V; i += 16) {
                    const float v = (float)x[i];
                    const uint64_t c = order_key(v, (uint32_t)i);
                    if (v > -INFINITY && c < last && c > k) k = c;
                }
                #pragma unroll
                for (int o = 8; o >= 1; o >>= 1) {
                    const uint64_t other = __shfl_xor(k, o);
                    k = other > k ? other : k;
                }
                if (l == 0) best[slot][kept] = k;     // 0: the row has no more
                last = k;
            }
            row_sync<1>();
        }
        if (there && l < g.n_top) {
            const bool good = s == s;
            const uint64_t k = good ? best[slot][l] : 0;
            const size_t o = (size_t)row * g.n_top + l;
            const float lp = (key_value(k) - base) - ln_s;
            g.top_logprob[o] = k ? (lp > 0.0f ? 0.0f : lp) : good ? -INFINITY : NAN;
            g.top_token[o] = k ? (int32_t)key_index(k) : -1;
        }
    }
}

template <typename T, int U>
void launch_short(const ScoreArgs& g, hipStream_t s) {
    const int grid = (g.N - 1) / 16 + 1;
    if (g.n_top) scores_short_kernel<T, U, true><<<grid, 256, 0, s>>>(g);
    else scores_short_kernel<T, U, false><<<grid, 256, 0, s>>>(g);
}

template <typename T, int W, int U>
void launch(const ScoreArgs& g, hipStream_t s) {
    constexpr int rows = W > 1 ? 1 : 4, threads = W > 1 ? 64 * W : 256;
    const int grid = (g.N - 1) / rows + 1;
    if (g.n_top) scores_kernel<T, W, U, true><<<grid, threads, 0, s>>>(g);
    else scores_kernel<T, W, U, false><<<grid, threads, 0, s>>>(g);
}

// Threads by the length of a row, which alone (with n_top) also fixes its order of
// sums. us on MI355X:
//   to 512, n_top <= 8: 16 lanes a row. 100000 x 256 fp32, 3 top 22, by a wave 55;
//     fp16, 8 top 26 and 67. More top tokens need the wave's 64 maxima.
//   to 64 CH: a wave with one chunk a lane, here for n_top > 8 only: 100000 x 256
//     fp16, 20 top 95, with four 127; 100000 x 512 93 and 126.
//   to 128 CH, 256 CH: a wave with two, four chunks a lane, the row in registers.
//     30000 x 1000 fp16 16.9 with two, 22.4 with four, 40 by two waves that walk it.
//   to 1024 CH, 4096 CH and above: 2, 4 and 8 waves that walk the row. 2 / 4 / 8:
//     10000 x 4000 fp16 17.1 / 28.3 / 52.0, 8000 x 8000 26.2 / 25.4 / 45.7, 4000 x 16000
//     28.3 / 28.0 / 24.9, 8192 x 50277 153 / 149 / 143 (16 waves: 194), 300 x 50277
//     20.5 / 13.1 / 12.1; fp32 8000 x 8000 48.8 / 47.5 / 42.5, 8192 x 50277 282 / 274 /
//     269.
template <typename T>
void launch_by_width(const ScoreArgs& g, hipStream_t s) {
    constexpr int CH = Chunk<T>::n;
    if (g.V <= 256 && g.n_top <= 8) launch_short<T, 16 / CH>(g, s);
    else if (g.V <= 512 && g.n_top <= 8) launch_short<T, 32 / CH>(g, s);
    else if (g.V <= 64 * CH) scores_kernel<T, 1, 1, true><<<(g.N - 1) / 4 + 1, 256, 0, s>>>(g);
    else if (g.V <= 128 * CH) launch<T, 1, 2>(g, s);
    else if (g.V <= 256 * CH) launch<T, 1, 4>(g, s);
    else if (g.V <= 1024 * CH) launch<T, 2, 4>(g, s);
    else if (g.V <= 4096 * CH) launch<T, 4, 4>(g, s);
    else launch<T, 8, 4>(g, s);
}

}  // namespace

extern "C" int kr_token_scores(const void* logits, int logits_f32, int N, int V, long long ld,
                               const int32_t* tokens, float* logprob, float* entropy, int n_top,
                               float* top_logprob, int32_t* top_token, void* stream) {
    KR_REQUIRE(N >= 0 && N <= 1 << 24, "kr_token_scores: N=%d must be in 0..%d", N, 1 << 24);
    KR_REQUIRE(V >= 1 && V <= 1 << 30 && ld >= V, "kr_token_scores: V=%d, ld=%lld", V, ld);
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
