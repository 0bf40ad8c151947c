// Products with weights in 4 bits, and the cast that makes them.
//
//   y[m, n] = sum_g scale[n, g] * sum_{k in group g} x[m, k] * e2m1(codes[n, k])  (+ bias[n]), rounded once to bf16
// codes [N, K / 2], two E2M1 values a byte, the even k in the low nibble; scales bf16 [N, K / G], G = 32, 64 or 128; x bf16.  That is how
// such weights are stored, and they are read as they are stored.
//
// For a few rows this reads weights and does little else: half a byte a weight, plus 2 / G of its scale.  The codes go to bf16 by the
// hardware's conversion (exact: 1 bit of mantissa), the products of a group to the fp32 accumulators of V_MFMA_F32_16X16X32_BF16 and from
// there times the group's scale, in fp32, onto the sums: nothing is rounded before the end.
//
// A wave works on 16 * NT columns of the output and 16 * MT rows; the waves of a block share K in chunks of 256 and are added up through LDS in
// wave order.  A lane reads 16 bytes of a row of codes: 32 weights in order, of one group of 32 at most.  What the MFMA multiplies in one
// instruction is 8 weights of each of the four lanes of a column, so for groups shorter than 128 the four lanes exchange their dwords
// first (four swaps of half and quarter waves for 32 weights); with groups of 128 the order of k inside a group does not matter.
#include "common.h"

#pragma clang fp contract(off)

namespace odl {
namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int kChunk = 256;                      // k of a wave and trip: whole 128-byte lines of codes

// eight codes of a dword -> eight bf16
__device__ __forceinline__ bf16x8 widen_codes(uint32_t w) {
    const uint32_t o[4] = {__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, 1.0f, 0)),
                           __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, 1.0f, 1)),
                           __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, 1.0f, 2)),
                           __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, 1.0f, 3))};
    return __builtin_bit_cast(bf16x8, u32x4{o[0], o[1], o[2], o[3]});
}

// Lanes l, l ^ 16, l ^ 32, l ^ 48 hold four dwords each: dword s of lane quarter q becomes dword q of quarter s.
__device__ __forceinline__ u32x4 exchange(u32x4 r) {
    auto a = __builtin_amdgcn_permlane32_swap(r.x, r.z, false, false);
    auto b = __builtin_amdgcn_permlane32_swap(r.y, r.w, false, false);
    auto lo = __builtin_amdgcn_permlane16_swap(a[0], b[0], false, false);
    auto hi = __builtin_amdgcn_permlane16_swap(a[1], b[1], false, false);
    return u32x4{lo[0], lo[1], hi[0], hi[1]};
}

struct Fp4Args {
    const uint16_t *x, *scales;
    const uint8_t *codes;
    const void *bias;
    uint16_t *y;
    int64_t M, N, K, ldx;
    int bias_f32;
};

template <int G, int MT, int NT, int WAVES>
__global__ __launch_bounds__(WAVES *kWave) void fp4_linear_kernel(const Fp4Args a) {
    constexpr int kGroups = kChunk / G;          // groups of a chunk
    __shared__ f32x4 part[WAVES][MT * NT][kWave];
    const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave, col = lane % 16, quarter = lane / 16;
    const int64_t n0 = (int64_t)blockIdx.x * (16 * NT), m0 = (int64_t)blockIdx.y * (16 * MT);
    const int64_t groups = a.K / G, chunks = (a.K + kChunk - 1) / kChunk;
    f32x4 acc[MT][NT];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[i][j] = f32x4{0, 0, 0, 0};

    u32x4 codes[NT][2];
    uint16_t scales[NT][kGroups];
    auto fetch = [&](int64_t ch) {
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            const int64_t n = n0 + 16 * j + col;
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const int64_t k = ch * kChunk + t * 128 + quarter * 32;
                codes[j][t] = n < a.N && k < a.K ? *reinterpret_cast<const u32x4 *>(a.codes + (n * a.K + k) / 2) : u32x4{0, 0, 0, 0};
            }
            const uint16_t *s = a.scales + n * groups + ch * kGroups;
            if ((ch + 1) * kChunk <= a.K) {      // (the same for every lane)
                if (n < a.N) __builtin_memcpy(scales[j], s, sizeof(scales[j]));
            } else {
#pragma unroll
                for (int g = 0; g < kGroups; ++g) scales[j][g] = n < a.N && ch * kGroups + g < groups ? s[g] : (uint16_t)0;
            }
            if (n >= a.N)
#pragma unroll
                for (int g = 0; g < kGroups; ++g) scales[j][g] = 0;
        }
    };
    if (wave < chunks) fetch(wave);
    for (int64_t ch = wave; ch < chunks; ch += WAVES) {
        u32x4 now[NT][2];
        float sc[NT][kGroups];
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            now[j][0] = codes[j][0];
            now[j][1] = codes[j][1];
#pragma unroll
            for (int g = 0; g < kGroups; ++g) sc[j][g] = bits_to_float((uint32_t)scales[j][g] << 16);
        }
        bf16x8 xf[2][MT][4];
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int s = 0; s < 4; ++s) {
                    const int64_t m = m0 + 16 * i + col;
                    const int64_t k = ch * kChunk + t * 128 + (G < 128 ? s * 32 + quarter * 8 : quarter * 32 + s * 8);
                    u32x4 v = {0, 0, 0, 0};
                    if (m < a.M && k < a.K) v = *reinterpret_cast<const u32x4 *>(a.x + m * a.ldx + k);
                    xf[t][i][s] = __builtin_bit_cast(bf16x8, v);
                }
        if (ch + WAVES < chunks) fetch(ch + WAVES);
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            constexpr int kSteps = G / 32;       // instructions of a group
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                const u32x4 w = G < 128 ? exchange(now[j][t]) : now[j][t];
                f32x4 p[MT];
#pragma unroll
                for (int s = 0; s < 4; ++s) {
                    const bf16x8 b = widen_codes(w[s]);
#pragma unroll
                    for (int i = 0; i < MT; ++i) {
                        const f32x4 from = s % kSteps == 0 ? f32x4{0, 0, 0, 0} : p[i];
                        p[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(xf[t][i][s], b, from, 0, 0, 0);
                        if (s % kSteps == kSteps - 1)
#pragma unroll
                            for (int e = 0; e < 4; ++e) acc[i][j][e] = __fmaf_rn(sc[j][(t * 4 + s) / kSteps], p[i][e], acc[i][j][e]);
                    }
                }
            }
        }
    }
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) part[wave][i * NT + j][lane] = acc[i][j];
    __syncthreads();
    for (int o = threadIdx.x; o < MT * NT * kWave; o += WAVES * kWave) {
        const int tile = o / kWave, l = o % kWave;
        f32x4 s = part[0][tile][l];
#pragma unroll
        for (int w = 1; w < WAVES; ++w) s += part[w][tile][l];
        const int64_t n = n0 + 16 * (tile % NT) + l % 16, m = m0 + 16 * (tile / NT) + l / 16 * 4;
        if (n < a.N) {
            float b = 0.0f;
            if (a.bias) b = a.bias_f32 ? reinterpret_cast<const float *>(a.bias)[n] : bits_to_float((uint32_t)reinterpret_cast<const uint16_t *>(a.bias)[n] << 16);
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (m + e < a.M) a.y[(m + e) * a.N + n] = (uint16_t)pack_bf16x2(a.bias ? s[e] + b : s[e], 0.0f);
        }
    }
}

// Weights to codes.  A group's scale is the bf16 nearest to max|w| / 6 (6 is the largest E2M1); a code is the E2M1 nearest to w / scale, ties to
// the even one, found by comparing |w| with the middles times the scale, which are exact products in fp32 (8 bits times 3).
// A lane holds 8 weights, G / 8 lanes a group.
template <int SRC, int G>
__global__ __launch_bounds__(256) void fp4_quantise_kernel(const void *__restrict__ w, int64_t lanes, uint32_t *__restrict__ codes,
                                                           uint16_t *__restrict__ scales) {
    constexpr int kLanes = G / 8;
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    float f[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = 0.0f;
    if (i < lanes) {
        if constexpr (SRC == ODL_BF16) {
            const u32x4 r = reinterpret_cast<const u32x4 *>(w)[i];
#pragma unroll
            for (int q = 0; q < 4; ++q) { f[2 * q] = bf16_lo(r[q]); f[2 * q + 1] = bf16_hi(r[q]); }
        } else {
            const float4 r0 = reinterpret_cast<const float4 *>(w)[2 * i], r1 = reinterpret_cast<const float4 *>(w)[2 * i + 1];
            f[0] = r0.x; f[1] = r0.y; f[2] = r0.z; f[3] = r0.w; f[4] = r1.x; f[5] = r1.y; f[6] = r1.z; f[7] = r1.w;
        }
    }
    uint32_t am = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) am = max(am, float_to_bits(f[e]) & 0x7fffffffu);
#pragma unroll
    for (int off = kLanes / 2; off > 0; off >>= 1) am = max(am, (uint32_t)__shfl_xor((int)am, off, kWave));
    const float most = bits_to_float(am), ratio = __fdiv_rn(most, 6.0f);
    uint32_t sb = f32_to_bf16_bits(ratio);
    if ((float_to_bits(ratio) & 0xffffu) == 0x8000u) {           // the rounded ratio lies between two bf16: which side the ratio itself lies on decides
        const float off = __fmaf_rn(ratio, 6.0f, -most);         // (exact)
        const uint32_t below = float_to_bits(ratio) >> 16;
        if (off != 0.0f) sb = off < 0.0f ? below + 1 : below;
    }
    const float s = bits_to_float(sb << 16);
    uint32_t word = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const float v = __builtin_fabsf(f[e]);
        // a middle belongs to the even of its two neighbours
        uint32_t code = (uint32_t)(v > 0.25f * s) + (uint32_t)(v >= 0.75f * s) + (uint32_t)(v > 1.25f * s) + (uint32_t)(v >= 1.75f * s) +
                        (uint32_t)(v > 2.5f * s) + (uint32_t)(v >= 3.5f * s) + (uint32_t)(v > 5.0f * s);
        if (s == 0.0f) code = 0;
        word |= (code | (float_to_bits(f[e]) >> 31 << 3)) << (4 * e);
    }
    if (i < lanes) {
        codes[i] = word;
        if (threadIdx.x % kLanes == 0) scales[i / kLanes] = (uint16_t)sb;
    }
}

bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
bool group_known(int group) { return group == 32 || group == 64 || group == 128; }

template <int G>
void launch_linear(const Fp4Args &a, hipStream_t stream) {
#define ODL_FP4(MT, NT, WAVES)                                                                                                              \
    hipLaunchKernelGGL((fp4_linear_kernel<G, MT, NT, WAVES>), dim3((unsigned)((a.N + 16 * NT - 1) / (16 * NT)), (unsigned)((a.M + 16 * MT - 1) / (16 * MT))), \
                       dim3(WAVES * kWave), 0, stream, a)
    if (a.M <= 16) ODL_FP4(1, 1, 8);
    else ODL_FP4(2, 1, 8);
#undef ODL_FP4
}

}  // namespace
}  // namespace odl

using namespace odl;

extern "C" int odl_fp8_fp4_linear(const void *x, int64_t ldx, const uint8_t *codes, const void *scales, int group, const void *bias, int bias_dtype,
                                  int64_t M, int64_t N, int64_t K, void *y, odl_stream_t stream_) {
    hipStream_t stream = reinterpret_cast<hipStream_t>(stream_);
    if (M < 0 || N < 0 || K < 0) return set_error(ODL_ERR_ARG, "odl_fp8_fp4_linear: negative shape");
    if (!group_known(group)) return set_error(ODL_ERR_ARG, "odl_fp8_fp4_linear: group %d (32, 64 or 128)", group);
    if (bias && bias_dtype != ODL_BF16 && bias_dtype != ODL_F32) return set_error(ODL_ERR_ARG, "odl_fp8_fp4_linear: bias_dtype %d", bias_dtype);
    if (K < group || K % group != 0) return set_error(ODL_ERR_SHAPE, "odl_fp8_fp4_linear: K must be a multiple of the group");
    if (M == 0 || N == 0) return ODL_OK;
    if (!x || !codes || !scales || !y) return set_error(ODL_ERR_ARG, "odl_fp8_fp4_linear: null pointer");
    if (ldx % 8 != 0 || (M > 1 && ldx < K) || !aligned16(x) || !aligned16(codes))
        return set_error(ODL_ERR_SHAPE, "odl_fp8_fp4_linear: x and codes must be 16-byte aligned, rows of x too");
    if (N > (int64_t)1 << 24 || M > (int64_t)1 << 20) return set_error(ODL_ERR_SHAPE, "odl_fp8_fp4_linear: up to 2^24 columns and 2^20 rows");
    Fp4Args a = {};
    a.x = static_cast<const uint16_t *>(x); a.scales = static_cast<const uint16_t *>(scales); a.codes = codes; a.bias = bias; a.y = static_cast<uint16_t *>(y);
    a.M = M; a.N = N; a.K = K; a.ldx = ldx; a.bias_f32 = bias_dtype == ODL_F32;
    if (group == 32) launch_linear<32>(a, stream);
    else if (group == 64) launch_linear<64>(a, stream);
    else launch_linear<128>(a, stream);
    return check_launch("odl_fp8_fp4_linear");
}

extern "C" int odl_fp8_fp4_quantise(const void *w, int src_dtype, int64_t N, int64_t K, int group, uint8_t *codes, void *scales, odl_stream_t stream_) {
    hipStream_t stream = reinterpret_cast<hipStream_t>(stream_);
    if (N < 0 || K < 0) return set_error(ODL_ERR_ARG, "odl_fp8_fp4_quantise: negative shape");
    if (src_dtype != ODL_BF16 && src_dtype != ODL_F32) return set_error(ODL_ERR_ARG, "odl_fp8_fp4_quantise: src_dtype %d", src_dtype);
    if (!group_known(group)) return set_error(ODL_ERR_ARG, "odl_fp8_fp4_quantise: group %d (32, 64 or 128)", group);
    if (K < group || K % group != 0) return set_error(ODL_ERR_SHAPE, "odl_fp8_fp4_quantise: K must be a multiple of the group");
    if (N == 0) return ODL_OK;
    if (!w || !codes || !scales) return set_error(ODL_ERR_ARG, "odl_fp8_fp4_quantise: null pointer");
    if (!aligned16(w) || !aligned16(codes)) return set_error(ODL_ERR_SHAPE, "odl_fp8_fp4_quantise: w and codes must be 16-byte aligned");
    const int64_t lanes = N * (K / 8), blocks = (lanes + 255) / 256;
    if (blocks >= 1 << 24) return set_error(ODL_ERR_SHAPE, "odl_fp8_fp4_quantise: %lld x %lld is too large", (long long)N, (long long)K);
#define ODL_FP4Q(SRC, G)                                                                                                                    \
    hipLaunchKernelGGL((fp4_quantise_kernel<SRC, G>), dim3((unsigned)blocks), dim3(256), 0, stream, w, lanes, reinterpret_cast<uint32_t *>(codes), \
                       static_cast<uint16_t *>(scales))
#define ODL_FP4Q_SRC(G) do { if (src_dtype == ODL_BF16) ODL_FP4Q(ODL_BF16, G); else ODL_FP4Q(ODL_F32, G); } while (0)
    if (group == 32) ODL_FP4Q_SRC(32);
    else if (group == 64) ODL_FP4Q_SRC(64);
    else ODL_FP4Q_SRC(128);
#undef ODL_FP4Q_SRC
#undef ODL_FP4Q
    return check_launch("odl_fp8_fp4_quantise");
}
