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
// Two kernels.  Thin, for a few rows: a block has 16 columns, its waves share K in chunks of 256 and are added up through LDS in wave order;
// 29 MB of codes for one token in 9.1 us (3.3 TB/s).  Wide, for more: a block has 128 columns and 16 to 128 rows, or 256 and 128, its waves share x in
// LDS, K is cut into runs where there are few blocks.
// In both a lane reads 16 bytes of a row of codes: 32 weights in order, of one group of 32 at most.  What the MFMA multiplies in one
// instruction is 8 weights of each of the four lanes of a column, so for groups shorter than 128 the four lanes exchange their dwords first (four
// swaps of half and quarter waves for 32 weights); with groups of 128 the order of k inside a group does not matter.
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
    float *partial;                              // [runs][M][N] where K is cut into runs of several blocks
    int64_t M, N, K, ldx;
    int bias_f32;
};

__device__ __forceinline__ float bias_of(const Fp4Args &a, int64_t n) {
    if (!a.bias) return 0.0f;
    return a.bias_f32 ? reinterpret_cast<const float *>(a.bias)[n] : bits_to_float((uint32_t)reinterpret_cast<const uint16_t *>(a.bias)[n] << 16);
}

// What a block of the thin kernel reads through LDS: the scales of its columns, and x where it is small (XLDS).  Scales are fetched by the
// lanes of one column at a time otherwise, 16 lines of memory for 64 bytes; x in four times as many loads as the codes.  (One row, 4096 -> 14336:
// 12.2 us with both from memory, 10.2 so; without any x and scales, which is not the product, 9.3.)
struct Fp4Tile {
    int groups, whole, pitch, xpitch;            // groups of a row, whole chunks, elements of a staged row of scales and of x
};

template <int G>
__host__ __device__ inline Fp4Tile fp4_tile(int K) {
    Fp4Tile t;
    t.groups = K / G;
    t.whole = K / kChunk;
    t.pitch = ((t.whole + 1) * (kChunk / G) + 7) / 8 * 8 + 2;         // (an odd number of dwords: the 16 columns lie in different banks)
    t.xpitch = (t.whole + 1) * kChunk + 8;
    return t;
}

// Up to 16 * MT rows a block.  Rows and columns past the end are read as the last ones are and not stored, so that nothing is masked on
// the way; the K behind the last whole chunk is.  A wave asks for the codes of its next chunk behind the products of one, and for x (from memory) of the
// next half chunk in front of those of one.
template <int G, int MT, int WAVES, bool XLDS>
__global__ __launch_bounds__(WAVES *kWave) void fp4_thin_kernel(const Fp4Args a) {
    constexpr int kGroups = kChunk / G;          // groups of a chunk
    constexpr int kSteps = G / 32;               // instructions of a group
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), col = lane % 16, quarter = lane / 16;
    const int K = (int)a.K;
    const Fp4Tile tile = fp4_tile<G>(K);
    const int64_t n0 = (int64_t)blockIdx.x * 16, m0 = (int64_t)blockIdx.y * (16 * MT);
    const uint8_t *cbase = a.codes + n0 * (a.K / 2);
    const uint16_t *sbase = a.scales + n0 * tile.groups, *xbase = a.x + m0 * a.ldx;
    uint16_t *slds = reinterpret_cast<uint16_t *>(lds), *xlds = slds + 16 * tile.pitch;
    const uint32_t coff = (uint32_t)(min(n0 + col, a.N - 1) - n0) * (uint32_t)(K / 2) + quarter * 16;
    uint32_t xoff[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) {
        const uint32_t m = (uint32_t)(min(m0 + 16 * i + col, a.M - 1) - m0);
        xoff[i] = m * (uint32_t)(XLDS ? tile.xpitch : a.ldx) + quarter * (G < 128 ? 8 : 32);
    }

    f32x4 acc[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) acc[i] = f32x4{0, 0, 0, 0};

    u32x4 codes[2], xv[XLDS ? 1 : 2][MT][4];
    auto fetch = [&](int ch) {
#pragma unroll
        for (int t = 0; t < 2; ++t) codes[t] = *reinterpret_cast<const u32x4 *>(cbase + (uint32_t)(ch * (kChunk / 2) + t * 64) + coff);
    };
    auto fetch_x = [&](int t, int ch) {
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                const uint32_t k = ch * kChunk + t * 128 + s * (G < 128 ? 32 : 8);
                if constexpr (XLDS) xv[0][i][s] = *reinterpret_cast<const u32x4 *>(xlds + k + xoff[i]);
                else xv[t][i][s] = *reinterpret_cast<const u32x4 *>(xbase + k + xoff[i]);
            }
    };
    auto multiply = [&](int t, int ch) {
        const u32x4 w = G < 128 ? exchange(codes[t]) : codes[t];
        const uint16_t *sc = slds + col * tile.pitch + ch * kGroups;
        uint32_t pair = 0;
        f32x4 p[MT];
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            const bf16x8 b = widen_codes(w[s]);
            const int g = (t * 4 + s) / kSteps;
            if (s == 0 || (s % kSteps == 0 && g % 2 == 0)) pair = *reinterpret_cast<const uint32_t *>(sc + g / 2 * 2);
            const float scale = g % 2 ? bf16_hi(pair) : bf16_lo(pair);
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                const f32x4 from = s % kSteps == 0 ? f32x4{0, 0, 0, 0} : p[i];
                p[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, xv[XLDS ? 0 : t][i][s]), b, from, 0, 0, 0);
                if (s % kSteps == kSteps - 1)
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[i][e] = __fmaf_rn(scale, p[i][e], acc[i][e]);
            }
        }
    };
    const int first = wave, last = first < tile.whole ? first + (tile.whole - 1 - first) / WAVES * WAVES : 0;
    if (first < tile.whole) {
        fetch(first);
        if constexpr (!XLDS) fetch_x(0, first);
    }
    {                                            // rows of scales, eight at a time; groups and columns past the end are zero
        const int per = (tile.pitch - 2) / 8, have = tile.groups;
        for (int i = threadIdx.x; i < 16 * per; i += WAVES * kWave) {
            const int r = i / per, g = i % per * 8;
            u32x4 v = {0, 0, 0, 0};
            const uint16_t *from = sbase + (uint32_t)(r * tile.groups + g);
            if (n0 + r < a.N) {
                if (g + 8 <= have) __builtin_memcpy(&v, from, 16);
                else
                    for (int e = 0; e < 8; ++e)
                        if (g + e < have) v[e / 2] |= (uint32_t)from[e] << (e % 2 * 16);
            }
            uint32_t *to = reinterpret_cast<uint32_t *>(slds + r * tile.pitch + g);
            to[0] = v.x; to[1] = v.y; to[2] = v.z; to[3] = v.w;
        }
    }
    if constexpr (XLDS) {                        // rows of x, the K past the end zero
        const int rows = (int)min((int64_t)(16 * MT), a.M - m0), per = (tile.xpitch - 8) / 8;
        for (int i = threadIdx.x; i < rows * per; i += WAVES * kWave) {
            const int r = i / per, k = i % per * 8;
            u32x4 v = {0, 0, 0, 0};
            if (k < K) v = *reinterpret_cast<const u32x4 *>(xbase + (uint32_t)(r * (uint32_t)a.ldx + k));
            *reinterpret_cast<u32x4 *>(xlds + r * tile.xpitch + k) = v;
        }
    }
    __syncthreads();
    for (int ch = first; ch < tile.whole; ch += WAVES) {
        if constexpr (XLDS) fetch_x(0, ch);
        else fetch_x(1, ch);
        multiply(0, ch);
        if constexpr (XLDS) fetch_x(1, ch);
        else fetch_x(0, min(ch + WAVES, last));
        multiply(1, ch);
        fetch(min(ch + WAVES, last));            // (behind the last chunk that one, and not used)
    }
    if (K % kChunk && wave == tile.whole % WAVES) {      // the rest of K, shorter than a chunk
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const int k = tile.whole * kChunk + t * 128 + quarter * 32;
            codes[t] = k < K ? *reinterpret_cast<const u32x4 *>(cbase + (uint32_t)(tile.whole * (kChunk / 2) + t * 64) + coff) : u32x4{0, 0, 0, 0};
        }
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            if constexpr (XLDS) {
                fetch_x(t, tile.whole);
            } else {
#pragma unroll
                for (int i = 0; i < MT; ++i)
#pragma unroll
                    for (int s = 0; s < 4; ++s) {
                        const int k = tile.whole * kChunk + t * 128 + s * (G < 128 ? 32 : 8), from = k + quarter * (G < 128 ? 8 : 32);
                        xv[t][i][s] = from < K ? *reinterpret_cast<const u32x4 *>(xbase + (uint32_t)k + xoff[i]) : u32x4{0, 0, 0, 0};
                    }
            }
            multiply(t, tile.whole);
        }
    }
    __syncthreads();                             // what was staged has been read
    f32x4 *part = reinterpret_cast<f32x4 *>(lds);
#pragma unroll
    for (int i = 0; i < MT; ++i) part[(wave * MT + i) * kWave + lane] = acc[i];
    __syncthreads();
    for (int o = threadIdx.x; o < MT * kWave; o += WAVES * kWave) {
        const int t = o / kWave, l = o % kWave;
        f32x4 s = part[o];
#pragma unroll
        for (int w = 1; w < WAVES; ++w) s += part[w * MT * kWave + o];
        const int64_t n = n0 + l % 16, m = m0 + 16 * t + l / 16 * 4;
        if (n >= a.N) continue;
        const float b = bias_of(a, n);
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (m + e < a.M) a.y[(m + e) * a.N + n] = (uint16_t)pack_bf16x2(a.bias ? s[e] + b : s[e], 0.0f);
    }
}

template <int G, int MT, int WAVES, bool XLDS>
void launch_thin(const Fp4Args &a, hipStream_t stream) {
    const Fp4Tile t = fp4_tile<G>((int)a.K);
    const int64_t rows = a.M < 16 * MT ? a.M : 16 * MT;
    const int64_t staged = 2 * (16 * (int64_t)t.pitch + (XLDS ? rows * t.xpitch : 0)), sums = (int64_t)WAVES * MT * kWave * 16;
    hipLaunchKernelGGL((fp4_thin_kernel<G, MT, WAVES, XLDS>), dim3((unsigned)((a.N + 15) / 16), (unsigned)((a.M + 16 * MT - 1) / (16 * MT))),
                       dim3(WAVES * kWave), (size_t)(staged > sums ? staged : sums), stream, a);
}

// Up to 16 * MT rows, many of them: x goes through LDS in phases of kPhase k, double-buffered, and the sixteen waves of a block share it, 16 columns each of
// 16 * kSlots and one of SHARES parts of a phase.  Codes, scales and x of the next phase are on their way while the waves multiply.
// Forms that were tried on the way, us, each beside this one as it was then: eight waves of 32 columns, which read x from LDS half as often, 32 rows
// 14336 -> 4096 18.0 (15.9), 8192 -> 28672 38.7 (33.1), 120 rows of that 95 (90); x through registers on its way to LDS, 120 rows 8192 -> 28672 94.8 (85.8).
// 128 rows by 256 columns bring x to LDS half as often as 128 by 128, 512 rows 4096 -> 14336 77 (90); for 120 rows of 8192 -> 28672 they are too few
// blocks, 129 (90), unless K is cut in two, 79 (81).
// As it is: 120 rows 8192 -> 28672, groups of 64, 79 us a call with its join: 710 TFLOP/s, a large bf16 product 1235.  Twenty calls in a row take 77 each, without half
// of the products 62, without three of four scalings 71, without bringing x to LDS 70; 512 rows 4096 -> 14336 72, 46, 72 and 70: bound by the products.  32 rows
// 14336 -> 4096 15.3, 15.3, 14.5 and 14.2: by the latency of two phases, the second asked for behind the first one's arrival, and of the join.
template <int G, int MT, int SHARES>
struct Fp4Wide {
    static constexpr int kWaves = 16, kThreads = kWaves * kWave, kSlots = kWaves / SHARES, kColumns = 16 * kSlots;
    static constexpr int kPhase = MT >= 8 ? 256 : MT >= 4 ? 512 : 1024, kShare = kPhase / SHARES, kSteps = kShare / 128;
    static constexpr int kPieces = 16 * MT * kPhase / 8 / kThreads, kGroups = kShare / G, kPairs = (kGroups + 1) / 2;
    static constexpr int kStage = 16 * MT * kPhase;          // elements of a buffer
    static constexpr int kRow = kPhase / 8;                  // 16-byte pieces of a row
    static_assert(kPieces * kThreads * 8 == kStage, "the lanes' pieces are the buffer");
};

template <int G, int MT, int SHARES>
__global__ __launch_bounds__((Fp4Wide<G, MT, SHARES>::kThreads)) void fp4_wide_kernel(const Fp4Args a, int run_k, int runs) {
    typedef Fp4Wide<G, MT, SHARES> W;
    constexpr int kPer = G / 32;                // instructions of a group
    __shared__ __attribute__((aligned(1024))) uint16_t stage[2][W::kStage];
    const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), col = lane % 16, quarter = lane / 16;
    const int share = wave / W::kSlots, K = (int)a.K, groups = K / G;
    const int64_t n0 = (int64_t)blockIdx.x * W::kColumns + wave % W::kSlots * 16, m0 = (int64_t)blockIdx.y * (16 * MT);
    const int k0 = blockIdx.z * run_k, k1 = min(K, k0 + run_k);
    // (columns and rows past the end are the last ones and not stored)
    const int64_t nb = min(n0, a.N - 1);
    const uint32_t n = (uint32_t)min((int64_t)col, a.N - 1 - nb), coff = n * (uint32_t)(K / 2) + quarter * 16, soff = n * (uint32_t)groups;
    const uint8_t *cbase = a.codes + nb * (a.K / 2);
    const uint16_t *sbase = a.scales + nb * groups, *xbase = a.x + m0 * a.ldx;
    // x goes to LDS without passing registers: 64 lanes' pieces of 16 bytes land one behind the other, so what can be chosen is what a lane reads.  Place
    // s of row r holds piece s ^ (r % 16) of it: the 16 rows that are read at a time then lie in different banks.
    uint32_t xrow[W::kPieces];
    int xk[W::kPieces];
#pragma unroll
    for (int i = 0; i < W::kPieces; ++i) {
        const int place = i * W::kThreads + threadIdx.x, r = place / W::kRow;
        xrow[i] = (uint32_t)min((int64_t)r, a.M - 1 - m0) * (uint32_t)a.ldx;
        xk[i] = ((place % W::kRow) ^ (r % 16)) * 8;
    }
    int xread[4];                                // where a lane finds the four k of a step
#pragma unroll
    for (int s = 0; s < 4; ++s) xread[s] = col * W::kPhase + share * W::kShare + ((G < 128 ? s * 4 + quarter : quarter * 4 + s) ^ col) * 8;
    const uint32_t stage_at = (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) uint16_t *)stage[0];
    f32x4 acc[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) acc[i] = f32x4{0, 0, 0, 0};

    u32x4 next_codes[W::kSteps];
    uint32_t next_scales[W::kPairs];
    auto fetch = [&](int k) {
        const int kc = k + share * W::kShare;
#pragma unroll
        for (int s = 0; s < W::kSteps; ++s) next_codes[s] = *reinterpret_cast<const u32x4 *>(cbase + (uint32_t)(kc / 2 + s * 64) + coff);
        if constexpr (W::kGroups == 1) next_scales[0] = sbase[(uint32_t)(kc / G) + soff];
        else __builtin_memcpy(next_scales, sbase + (uint32_t)(kc / G) + soff, sizeof(next_scales));
    };
    auto fetch_end = [&](int k) {                            // a phase that k1 ends: what is behind it is zero
        const int kc = k + share * W::kShare;
#pragma unroll
        for (int s = 0; s < W::kSteps; ++s) {
            next_codes[s] = u32x4{0, 0, 0, 0};
            if (kc + s * 128 + quarter * 32 < k1) next_codes[s] = *reinterpret_cast<const u32x4 *>(cbase + (uint32_t)(kc / 2 + s * 64) + coff);
        }
        uint32_t v[2 * W::kPairs];                           // (all asked for before any is looked at)
#pragma unroll
        for (int g = 0; g < 2 * W::kPairs; ++g) v[g] = sbase[(uint32_t)min(kc / G + g, groups - 1) + soff];
#pragma unroll
        for (int g = 0; g < W::kPairs; ++g)
            next_scales[g] = (kc + 2 * g * G < k1 ? v[2 * g] : 0u) | (kc + (2 * g + 1) * G < k1 ? v[2 * g + 1] << 16 : 0u);
    };
    auto ask_for = [&](int to, int k) {
        if (k + W::kPhase <= k1) fetch(k);
        else fetch_end(k);
#pragma unroll
        for (int i = 0; i < W::kPieces; ++i) {               // (pieces behind k1: the last one, zeroed below)
            const uint16_t *from = xbase + xrow[i] + min(k + xk[i], k1 - 8);
            asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off"
                         ::"s"(stage_at + 2 * to * W::kStage + (i * W::kWaves + wave) * 1024), "v"(from) : "memory");
        }
    };
    auto arrived = [&](int to, int k) {                      // this lane's own pieces
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        if (k + W::kPhase <= k1) return;
#pragma unroll
        for (int i = 0; i < W::kPieces; ++i)
            if (k + xk[i] >= k1) *reinterpret_cast<u32x4 *>(stage[to] + (i * W::kThreads + threadIdx.x) * 8) = u32x4{0, 0, 0, 0};
    };
    ask_for(0, k0);
    arrived(0, k0);
    __syncthreads();
    int buf = 0;
    for (int k = k0; k < k1; k += W::kPhase, buf ^= 1) {
        u32x4 codes[W::kSteps];
        uint32_t scales[W::kPairs];
#pragma unroll
        for (int s = 0; s < W::kSteps; ++s) codes[s] = next_codes[s];
#pragma unroll
        for (int g = 0; g < W::kPairs; ++g) scales[g] = next_scales[g];
        const bool more = k + W::kPhase < k1;
        if (more) ask_for(buf ^ 1, k + W::kPhase);
        const uint16_t *xs = stage[buf];
        // Units of 16 rows and one group of k, software-pipelined: x is asked for kAhead units before its products, and the products of a
        // unit are scaled onto the sums behind the products of the next kBehind.
        constexpr int kUnits = W::kSteps * (4 / kPer) * MT, kAhead = 4 / kPer, kBehind = kPer > 2 ? 1 : 2;
        bf16x8 xq[kAhead + 1][kPer], b[kPer];
        f32x4 p[kBehind + 1];
        float scale[4];
        auto ask = [&](int u) {                  // (every index is known at compile time)
            const int i = u % MT, s0 = u / MT * kPer;
#pragma unroll
            for (int s = 0; s < kPer; ++s)
                xq[u % (kAhead + 1)][s] = __builtin_bit_cast(
                    bf16x8, *reinterpret_cast<const u32x4 *>(xs + xread[(s0 + s) % 4] + i * 16 * W::kPhase + (s0 + s) / 4 * 128));
        };
#pragma unroll
        for (int u = 0; u < (kAhead < kUnits ? kAhead : kUnits); ++u) ask(u);
        u32x4 w;
#pragma unroll
        for (int u = 0; u < kUnits + kBehind; ++u) {
            if (u + kAhead < kUnits) ask(u + kAhead);
            if (u < kUnits) {
                const int g = u / MT, s0 = g * kPer;
                if (u % MT == 0) {
                    if (s0 % 4 == 0) w = G < 128 ? exchange(codes[s0 / 4]) : codes[s0 / 4];
                    scale[g % 4] = g % 2 ? bf16_hi(scales[g / 2]) : bf16_lo(scales[g / 2]);
#pragma unroll
                    for (int s = 0; s < kPer; ++s) b[s] = widen_codes(w[(s0 + s) % 4]);
                }
                f32x4 &to = p[u % (kBehind + 1)];
#pragma unroll
                for (int s = 0; s < kPer; ++s)
                    to = __builtin_amdgcn_mfma_f32_16x16x32_bf16(xq[u % (kAhead + 1)][s], b[s], s == 0 ? f32x4{0, 0, 0, 0} : to, 0, 0, 0);
            }
            if (u >= kBehind) {
                const int v = u - kBehind, i = v % MT;
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[i][e] = __fmaf_rn(scale[v / MT % 4], p[v % (kBehind + 1)][e], acc[i][e]);
                asm volatile("" : "+v"(acc[i]));             // (not put off behind the loop, which would spill the products)
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        if (more) arrived(buf ^ 1, k + W::kPhase);
        __syncthreads();
    }
    if constexpr (SHARES == 2) {                 // the second share's sums onto the first's
        f32x4 *part = reinterpret_cast<f32x4 *>(stage[0]) + wave % W::kSlots * (MT * kWave) + lane;
        static_assert(sizeof(stage) >= W::kSlots * MT * kWave * sizeof(f32x4), "the sums fit into the stage");
        if (share) {
#pragma unroll
            for (int i = 0; i < MT; ++i) part[i * kWave] = acc[i];
        }
        __syncthreads();
        if (share) return;
#pragma unroll
        for (int i = 0; i < MT; ++i) acc[i] += part[i * kWave];
    }
    if (n0 + col >= a.N) return;
    const float bias = bias_of(a, n0 + col);
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int64_t m = m0 + 16 * i + quarter * 4 + e;
            if (m >= a.M) continue;
            if (runs > 1) a.partial[(blockIdx.z * a.M + m) * a.N + n0 + col] = acc[i][e];
            else a.y[m * a.N + n0 + col] = (uint16_t)pack_bf16x2(a.bias ? acc[i][e] + bias : acc[i][e], 0.0f);
        }
}

template <int G, int MT, int SHARES>
int launch_wide(const Fp4Args &a, int runs, hipStream_t stream) {
    typedef Fp4Wide<G, MT, SHARES> W;
    const int phase = W::kPhase, run_k = (int)((a.K + runs - 1) / runs + phase - 1) / phase * phase;
    runs = (int)((a.K + run_k - 1) / run_k);                 // (no run is empty)
    hipLaunchKernelGGL((fp4_wide_kernel<G, MT, SHARES>), dim3((unsigned)((a.N + W::kColumns - 1) / W::kColumns), (unsigned)((a.M + 16 * MT - 1) / (16 * MT)), (unsigned)runs),
                       dim3(W::kThreads), 0, stream, a, run_k, runs);
    return runs;
}

// Runs of K of several blocks, added in their order.
__global__ __launch_bounds__(256) void fp4_join_kernel(const Fp4Args a, int runs) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, total = a.M * a.N;
    if (i >= total) return;
    float s = 0.0f;
    for (int r = 0; r < runs; r += 8) {
        float v[8];                              // (eight on their way at once)
#pragma unroll
        for (int u = 0; u < 8; ++u) v[u] = r + u < runs ? a.partial[(r + u) * total + i] : 0.0f;
#pragma unroll
        for (int u = 0; u < 8; ++u) s += v[u];
    }
    if (a.bias) s += bias_of(a, i % a.N);
    a.y[i] = (uint16_t)pack_bf16x2(s, 0.0f);
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

// The thin kernel stages the scales of whole rows, which for a very long K do not fit, and up to 16 rows of x where they fit beside them: 4 rows
// 14336 -> 4096 13.6 -> 10.4 us, 16 rows 2048 -> 8192 9.5 -> 6.7.
constexpr int64_t kThinLds = 64 * 1024, kThinX = 150 * 1024;

template <int G>
bool x_in_lds(int64_t M, int64_t K) {
    const Fp4Tile t = fp4_tile<G>((int)K);
    return M <= 16 && 2 * (16 * (int64_t)t.pitch + M * t.xpitch) <= kThinX;
}

// How a product is done: rows of a block of the wide kernel in 16s (0: the thin kernel), in how many parts its waves share a phase, and runs of K.
struct Fp4Plan {
    int mt, shares, runs;
};

// The cheapest by what a block was measured to take, ns for each k: thin 0.30 + 0.055 a row with x in LDS, 0.39 + 0.058 a row without; wide 3.1, 3.7, 5.0 and
// 9.2 for 16, 32, 64 and 128 rows, 15 for 128 rows by 256 columns, and 1.3 to 4.6 us besides, with as many blocks at a time as there are compute
// units; a join 1.5 us and 0.86 ps for each number.  Thin blocks of more than four for each unit do not begin together: one row 8192 -> 28672 35 us, wide 29.
// Over 182 products of 5 to 2048 rows, 768 -> 768 to 28672 -> 8192, what this takes is 1.5 % off the best of them all on average and 24 % at worst, over
// 176 of 1 to 16 rows 1 and 32 %.  (By rows and size of the weights alone: 20 % and 95 %.  Blocks of 16 rows were timed for up to 48.)
template <int G>
Fp4Plan plan(int64_t M, int64_t N, int64_t K) {
    const bool fits = 2 * 16 * (int64_t)fp4_tile<G>((int)K).pitch <= kThinLds;
    const int64_t cus = device_cu_count(), thin = (N + 15) / 16 * (M <= 16 ? 1 : (M + 31) / 32), most = thin > cus ? thin : cus;
    Fp4Plan best = {0, 1, 1};
    int64_t least = !fits ? INT64_MAX : x_in_lds<G>(M, K) ? 3400000 + K * (300 + 55 * M) * most / cus : 4100000 + K * (390 + 58 * (M < 32 ? M : 32)) * most / cus;      // ps
    if (fits && thin > 4 * cus) least += least / 5 * 2;
    if (least < 6800000) return best;                        // (no wide one begins below)
    static constexpr struct { int mt, shares, phase, per_k, start; } kinds[] = {
        {1, 2, 1024, 3100, 1300000}, {2, 2, 1024, 3700, 1700000}, {4, 2, 512, 5000, 3000000}, {8, 2, 256, 9200, 4500000}, {8, 1, 256, 15000, 4600000}};
    for (const auto &kind : kinds) {
        if (kind.mt == 1 && M > 48) continue;
        const int64_t columns = 256 / kind.shares, tiles = (N + columns - 1) / columns * ((M + 16 * kind.mt - 1) / (16 * kind.mt));
        for (const int runs : {1, 2, 3, 4, 6, 8, 12, 16, 24, 32}) {
            if (runs > 1 && (runs * kind.phase > K || M * N >= (int64_t)1 << 32)) break;
            const int64_t k = ((K + runs - 1) / runs + kind.phase - 1) / kind.phase * kind.phase, rounds = (tiles * ((K + k - 1) / k) + cus - 1) / cus;
            const int64_t cost = 2400000 + rounds * (kind.start + k * kind.per_k) + (runs > 1 ? 1500000 + runs * M * N * 43 / 50 : 0);
            if (cost < least) { least = cost; best = {kind.mt, kind.shares, runs}; }
        }
    }
    return best;
}

template <int G>
void launch_linear(const Fp4Args &a, const Fp4Plan how, hipStream_t stream) {
    if (how.mt == 0) {
        const Fp4Tile t = fp4_tile<G>((int)a.K);
        const bool lds = x_in_lds<G>(a.M, a.K), deep = t.whole >= 32;
        // long rows: 16 waves share them (14336 -> 4096 11.5 -> 10.5, 4096 -> 14336 no faster)
        if (lds && deep) launch_thin<G, 1, 16, true>(a, stream);
        else if (lds) launch_thin<G, 1, 8, true>(a, stream);
        else if (a.M <= 16) launch_thin<G, 1, 8, false>(a, stream);
        else launch_thin<G, 2, 4, false>(a, stream);
        return;
    }
    int runs = how.runs;
    if (how.mt == 1) runs = launch_wide<G, 1, 2>(a, runs, stream);
    else if (how.mt == 2) runs = launch_wide<G, 2, 2>(a, runs, stream);
    else if (how.mt == 4) runs = launch_wide<G, 4, 2>(a, runs, stream);
    else if (how.shares == 2) runs = launch_wide<G, 8, 2>(a, runs, stream);
    else runs = launch_wide<G, 8, 1>(a, runs, stream);
    if (runs > 1) hipLaunchKernelGGL(fp4_join_kernel, dim3((unsigned)((a.M * a.N + 255) / 256)), dim3(256), 0, stream, a, runs);
}

Fp4Plan plan_of(int64_t M, int64_t N, int64_t K, int group) {
    return group == 32 ? plan<32>(M, N, K) : group == 64 ? plan<64>(M, N, K) : plan<128>(M, N, K);
}

}  // namespace
}  // namespace odl

using namespace odl;

// Partial results that a call writes: its workspace is as many times M * N floats; 0 needs none.
extern "C" int odl_fp8_fp4_linear_runs(int64_t M, int64_t N, int64_t K, int group) {
    if (M < 1 || N < 1 || K < 1 || M > (int64_t)1 << 20 || N > (int64_t)1 << 22 || K > (int64_t)1 << 24) return 0;
    const int runs = plan_of(M, N, K, group).runs;
    return runs > 1 ? runs : 0;
}

extern "C" int odl_fp8_fp4_linear(const void *x, int64_t ldx, const uint8_t *codes, const void *scales, int group, const void *bias, int bias_dtype,
                                  int64_t M, int64_t N, int64_t K, void *y, float *workspace, int64_t workspace_bytes, odl_stream_t stream_) {
    hipStream_t stream = reinterpret_cast<hipStream_t>(stream_);
    if (M < 0 || N < 0 || K < 0) return set_error(ODL_ERR_ARG, "odl_fp8_fp4_linear: negative shape");
    if (!group_known(group)) return set_error(ODL_ERR_ARG, "odl_fp8_fp4_linear: group %d (32, 64 or 128)", group);
    if (bias && bias_dtype != ODL_BF16 && bias_dtype != ODL_F32) return set_error(ODL_ERR_ARG, "odl_fp8_fp4_linear: bias_dtype %d", bias_dtype);
    if (K < group || K % group != 0) return set_error(ODL_ERR_SHAPE, "odl_fp8_fp4_linear: K must be a multiple of the group");
    if (M == 0 || N == 0) return ODL_OK;
    if (!x || !codes || !scales || !y) return set_error(ODL_ERR_ARG, "odl_fp8_fp4_linear: null pointer");
    if (ldx % 8 != 0 || (M > 1 && ldx < K) || ldx > (int64_t)1 << 24 || !aligned16(x) || !aligned16(codes))
        return set_error(ODL_ERR_SHAPE, "odl_fp8_fp4_linear: x and codes must be 16-byte aligned, rows of x too, at most 2^24 elements apart");
    if (N > (int64_t)1 << 22 || M > (int64_t)1 << 20 || K > (int64_t)1 << 24)
        return set_error(ODL_ERR_SHAPE, "odl_fp8_fp4_linear: up to 2^20 rows, 2^22 columns and 2^24 inputs");
    const Fp4Plan how = plan_of(M, N, K, group);
    if (how.runs > 1 && (!workspace || workspace_bytes / 4 / M / N < how.runs))
        return set_error(ODL_ERR_ARG, "odl_fp8_fp4_linear: a workspace of %d * M * N floats is needed", how.runs);
    Fp4Args a = {};
    a.x = static_cast<const uint16_t *>(x); a.scales = static_cast<const uint16_t *>(scales); a.codes = codes; a.bias = bias; a.y = static_cast<uint16_t *>(y);
    a.partial = workspace; a.M = M; a.N = N; a.K = K; a.ldx = M > 1 ? ldx : 0; a.bias_f32 = bias_dtype == ODL_F32;
    if (group == 32) launch_linear<32>(a, how, stream);
    else if (group == 64) launch_linear<64>(a, how, stream);
    else launch_linear<128>(a, how, stream);
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
