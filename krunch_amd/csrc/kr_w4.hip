// Products with 4-bit weights: x [M, K] fp16 times a [K, N] weight held as
// integers q in -8..7 with one fp16 scale per output channel and group of 32,
// 64 or 128 inputs (K % 32 == 0).
//
//   y[m, n] = sum_g s[g, n] * c_g,   c_g = sum_{k in group g} q[n, k] x[m, k]
//
// q x has at most 15 significant bits, so c_g is a chain of exact products on
// v_mfma_f32_16x16x32_f16 (k ascending, from zero), and the scale is applied in
// fp32. Reduction contract, whatever the kernel: slices of 512 inputs, in a
// slice P = fma(s_g, c_g, P) over its groups in order from zero, then y = P_0
// + P_1 + ... left to right; so a row has the same bits for any M.
//
// Layout (kr_w4_bytes): blocks of 16 outputs x 128 inputs, 1 KB, (N / 16) major
// and K / 128 minor. Lane l holds 4 words, word c the inputs 32 c + 8 (l / 16)
// .. + 7 of output l % 16, as the MFMA operand of k-step c: a wave's load of a
// block is one contiguous KB, 16 bytes a lane. Nibbles are q + 8, in the order
// 0, 2, 4, 6, 1, 3, 5, 7 from the low one up: two ANDs (bits 0..3 and 4..7 of
// each half) and one shift give fp16 pairs in operand order, by their place in
// the mantissa of 1024 and of 64, and one packed addition takes 1024 + 8 or
// 64 + 8 off, exactly: 9 operations for 8 weights. Padding is q = 0, scale 0.
#include "kr_gemm_epilogue.h"
#include "krunch_hip.h"

namespace {

constexpr int kBlockK = 128, kSliceK = 512;
constexpr int kMaxSplit = 8;                 // waves that share a tile's slices

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

// The 8 weights of a word as an MFMA operand.
__device__ __forceinline__ kr_half8 unpack(uint32_t w) {
    const kr_half2 k1024 = {(kr_half)-1032.0f, (kr_half)-1032.0f};
    const kr_half2 k64 = {(kr_half)-72.0f, (kr_half)-72.0f};
    const uint32_t v = w >> 8;
    const kr_half2 a = __builtin_bit_cast(kr_half2, (w & 0x000F000Fu) | 0x64006400u) + k1024;
    const kr_half2 b = __builtin_bit_cast(kr_half2, (w & 0x00F000F0u) | 0x54005400u) + k64;
    const kr_half2 c = __builtin_bit_cast(kr_half2, (v & 0x000F000Fu) | 0x64006400u) + k1024;
    const kr_half2 d = __builtin_bit_cast(kr_half2, (v & 0x00F000F0u) | 0x54005400u) + k64;
    return kr_half8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

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

__device__ __forceinline__ kr_float4 scale4(const kr_half* s) {
    const kr_half4 h = *reinterpret_cast<const kr_half4*>(s);
    return kr_float4{(float)h[0], (float)h[1], (float)h[2], (float)h[3]};
}

// One slice of one 16-output tile against MT x 16 rows, x read from memory.
// GS = k-steps per group.
template <int MT, int GS>
__device__ __forceinline__ void slice_rows(const W4Args& g, int tile, int k_begin, int k_end,
                                           const kr_half* const (&xr)[MT], kr_float4 (&P)[MT]) {
    const int lane = threadIdx.x & 63;
    const int kb_all = (g.o.K + kBlockK - 1) / kBlockK;
    const kr_int4* q = g.q + ((size_t)tile * kb_all + k_begin / kBlockK) * 64 + lane;
    const kr_half* sc = g.scales + (size_t)(k_begin / (32 * GS)) * g.n16 + 16 * tile + 4 * (lane >> 4);
    #pragma unroll
    for (int t = 0; t < MT; t++) P[t] = kr_float4{0, 0, 0, 0};
    for (int k0 = k_begin; k0 < k_end; k0 += kBlockK, q += 64) {
        const kr_int4 w = *q;
        kr_float4 c[MT];
        #pragma unroll
        for (int t = 0; t < MT; t++) c[t] = kr_float4{0, 0, 0, 0};
        #pragma unroll
        for (int i = 0; i < 4; i++) {
            const int k = k0 + 32 * i;
            if (k >= k_end) break;
            const kr_half8 a = unpack((uint32_t)w[i]);
            #pragma unroll
            for (int t = 0; t < MT; t++)
                c[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                    a, *reinterpret_cast<const kr_half8*>(xr[t] + k), c[t], 0, 0, 0);
            if ((i + 1) % GS == 0 || k + 32 >= k_end) {
                const kr_float4 s = scale4(sc);
                sc += g.n16;
                #pragma unroll
                for (int t = 0; t < MT; t++) {
                    #pragma unroll
                    for (int r = 0; r < 4; r++) P[t][r] = __builtin_fmaf(s[r], c[t][r], P[t][r]);
                    c[t] = kr_float4{0, 0, 0, 0};
                }
            }
        }
    }
}

// Few rows: a wave has a 16-output tile against up to 16 MT rows. With SPLIT,
// the workgroup's waves share one tile, wave w its slices w, w + waves, ...,
// joined in LDS in slice order; else each wave has a tile of its own.
template <int MT, int GS, int EP, bool SPLIT>
__global__ void __launch_bounds__(SPLIT ? 64 * kMaxSplit : 256) w4_rows_kernel(W4Args g) {
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
    const int tile = SPLIT ? blockIdx.x : blockIdx.x * waves + wave;
    const int m0 = blockIdx.y * 16 * MT;
    if (!SPLIT && 16 * tile >= g.n16) return;
    const kr_half* xr[MT];
    #pragma unroll
    for (int t = 0; t < MT; t++) {
        const int m = m0 + 16 * t + (lane & 15);       // rows past M read the last one
        xr[t] = g.x + (size_t)(m < g.o.M ? m : g.o.M - 1) * g.ldx + 8 * (lane >> 4);
    }
    const int slices = (g.o.K + kSliceK - 1) / kSliceK;
    kr_float4 total[MT], P[MT];
    if constexpr (SPLIT) {
        extern __shared__ kr_float4 part[];           // [slices][MT][64]
        for (int z = wave; z < slices; z += waves) {
            const int k1 = (z + 1) * kSliceK < g.o.K ? (z + 1) * kSliceK : g.o.K;
            slice_rows<MT, GS>(g, tile, z * kSliceK, k1, xr, P);
            #pragma unroll
            for (int t = 0; t < MT; t++) part[(z * MT + t) * 64 + lane] = P[t];
        }
        __syncthreads();
        for (int t = wave; t < MT; t += waves) {
            kr_float4 y = part[t * 64 + lane];
            for (int z = 1; z < slices; z++) y += part[(z * MT + t) * 64 + lane];
            store4<EP>(g.o, m0 + 16 * t + (lane & 15), 16 * tile + 4 * (lane >> 4), y);
        }
    } else {
        for (int z = 0; z < slices; z++) {
            const int k1 = (z + 1) * kSliceK < g.o.K ? (z + 1) * kSliceK : g.o.K;
            slice_rows<MT, GS>(g, tile, z * kSliceK, k1, xr, P);
            #pragma unroll
            for (int t = 0; t < MT; t++) total[t] = z == 0 ? P[t] : total[t] + P[t];
        }
        #pragma unroll
        for (int t = 0; t < MT; t++)
            store4<EP>(g.o, m0 + 16 * t + (lane & 15), 16 * tile + 4 * (lane >> 4), total[t]);
    }
}

template <int MT, int GS, int EP>
int launch_rows(const W4Args& g, hipStream_t s) {
    const int tiles = g.n16 / 16, slices = (g.o.K + kSliceK - 1) / kSliceK;
    const int mt = (g.o.M + 16 * MT - 1) / (16 * MT);
    const size_t lds = (size_t)slices * MT * 64 * sizeof(kr_float4);
    if (slices > 1 && (long long)tiles * mt < 1024 && lds <= 65536) {
        const int waves = slices < kMaxSplit ? slices : kMaxSplit;
        w4_rows_kernel<MT, GS, EP, true><<<dim3(tiles, mt), 64 * waves, lds, s>>>(g);
    } else {
        w4_rows_kernel<MT, GS, EP, false><<<dim3((tiles + 3) / 4, mt), 256, 0, s>>>(g);
    }
    KR_LAUNCHED();
    return KR_OK;
}

template <int GS, int EP>
int launch_by_rows(const W4Args& g, hipStream_t s) {
    if (g.o.M <= 16) return launch_rows<1, GS, EP>(g, s);
    if (g.o.M <= 32) return launch_rows<2, GS, EP>(g, s);
    return launch_rows<4, GS, EP>(g, s);
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
// W[k * ldk + n * ldn]; one of the two is 1 in use.
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
    KR_REQUIRE(K >= 32 && K % 32 == 0 && K <= (1 << 24), "%s: K=%d must be a multiple of 32", who, K);
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
