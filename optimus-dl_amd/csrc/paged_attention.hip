// Attention of a step's new tokens over a paged cache that holds them.  For a row (token, head) at position p, with the keys and values of its group:
//   s_i = scale * q . k_i  (softcap * tanh(s_i / softcap)),  out = sum_i 2^(c s_i - m) v_i / sum_i 2^(c s_i - m),  c = log2 e, i the keys that the row sees
// in one pass over the keys, with a running maximum m and sum.  Heads of a group share keys, so what a matrix instruction takes as its other operand
// is the rows (token, head of the group) of one key head: S^T = K Q^T and O^T = V^T P^T by V_MFMA_F32_32X32X16_BF16.  In the result of the first a
// lane holds one row's scores for 16 of 32 keys: sums and maxima of a row are a lane's own but for one exchange with lane ^ 32, and those registers are
// the second operand of the second product as they are, when V^T's keys are taken in the same order (ds_read_b64_tr_b16 fetches them so).
//
// Two kernels.  Few rows a key head (32 at most: single tokens, drafts): the cache is read once and that bounds it; the four waves of a block take
// every fourth tile of 32 keys, each on its own, and are joined in LDS.  Many (prompts, chunks): MFMA and the exponentials bound it; eight waves of 32
// rows share tiles of 64 keys, three in LDS.  In both tiles of bf16 go to LDS without passing registers, one or two ahead, and where there are fewer
// tiles of rows than compute units the keys are cut into splits, whose sums a third kernel joins in order.  Every block works out from the lengths which
// part is its own (`find`): lengths never pass the host.
//
// Measured (calls in a row, host included; a large copy moves 5.1 TB/s on this card, a large product in bf16 makes 1206 TFLOP/s):
//   few   64 sequences of up to 8192 tokens, 32 heads on 8 of 128, bf16               298 us   5.4 TB/s  (E4M3 191, 4.2: codes pass registers)
//         1 sequence of 131072 tokens, the same heads                                 110 us   4.9 TB/s  (of which the join 5 to 10; E4M3 71)
//         32 sequences of 4099, 5 new tokens of each, E4M3                             69 us   3.9 TB/s  (the join 10; bf16 110)
//   many  2048 new tokens behind 14336, 32 heads on 8 of 128                          497 us   1037 TFLOP/s  (the card runs at some 2.0 GHz meanwhile; E4M3 564, capped 670)
//         12 prompts of up to 1000 tokens behind up to 3000, 16 heads on 4 of 96, capped, a window of 1500: 171 us  (288 tiles on 256 compute units: two rounds; without the cap 128)
// A sequence with up to 32 rows a key head fills one tile of the first kernel; from there on that would read the cache again for every 32 rows.
#include "paged.h"

#pragma clang fp contract(off)

namespace odl {
namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __attribute__((address_space(3))) uint8_t lds_u8;

constexpr int kFewRows = 32, kFewKeys = 32, kFewWaves = 4;
constexpr int kManyRows = 256, kManyKeys = 64, kManyWaves = 8;
// Blocks that splits are made for: as many as run at a time.  Of the large ones that is one a compute unit (with 256 / 512 the chunk takes 524 / 556, the prompts 206 / 231).
// Of the small ones LDS decides: two, and one of those that hold two stages of bf16 for heads above 64 (with 512 / 256 for these: one token behind 131071 124 / 115 us, 32 sequences of
// 4099 with 5 new tokens 122 / 114, 8 of 1000 24 / 18, 64 of 8192 435 / 435, all with 32 heads on 8 of 128).
constexpr int few_lds(int D, bool e4m3) {
    const int tiles = kFewWaves * (e4m3 ? 1 : 2) * 2 * kFewKeys * 2 * D, joined = kFewWaves * 32 * (D + 4) * 4 + kFewWaves * 32 * 8;
    return tiles > joined ? tiles : joined;
}
constexpr int kManyTarget = 256;
constexpr int few_target(int D, bool e4m3) { return few_lds(D, e4m3) <= 80 * 1024 ? 512 : 256; }
// Steps of 128 keys that a split of the small ones has at least.  A table of up to four is not cut, which saves the join.  Behind a wider one the join is launched, whatever the lengths
// are, and the longest sequence decides: up to two steps stay whole, up to sixteen are cut into single ones, more into two at least, since a join takes longer the more
// there is to join.  One token behind 200 / 500 / 1000 / 4000 in a table of 4096 (a captured step, us): 12 heads of 64 10.8 / 11.7 / 11.9 / 13.9, with one step everywhere 11.4 / 11.6 / 11.9 /
// 14.9, with two 10.8 / 12.5 / 12.6 / 13.9; 32 heads on 8 of 128 12.8 / 13.3 / 13.5 / 15.5, 12.8 / 13.0 / 13.3 / 16.3 and 12.9 / 14.5 / 14.7 / 15.5.
constexpr int kUncut = 4, kWhole = 2, kSingle = 16;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kSlack = 8.0f;                                 // how far, in powers of two, a running maximum may lag behind

// What lanes read that have no key: a row of zeros.
__device__ const uint32_t g_zeros[64] __attribute__((aligned(256))) = {};

struct Attend {
    Paged p;
    const uint16_t *q;
    int64_t q_row, q_head;
    int heads, group, window;                                  // group: heads of a key head; window: INT_MAX for none
    int least_rows, most_rows;                                 // rows a key head of the sequences that this launch is for
    float scale, softcap;
    uint16_t *out;
    float *partial;                                            // [slots][rows of a tile][D] sums, then [slots][rows of a tile][2] maxima and sums
    int64_t slots;
};

// ---------------------------------------------------------------------------------------------------------------- whose work a block does
// A sequence's share: `tiles` of rows, each cut into `splits` of its keys.
struct Share {
    Run run;
    int length;                                                // tokens in the cache, within the table's reach
    uint32_t tiles, units, splits;
};

template <int ROWS, int KEYS>
__device__ __forceinline__ Share share_of(const Attend &a, int s) {
    Share h = {{0, 0}, 0, 0, 0, 0};
    if (s >= a.p.seqs) return h;
    h.run = run_of(a.p, s);
    h.length = a.p.lengths[s];
    const int rows = h.run.n * a.group, held = min(max(h.length, 0), a.p.reach);
    if (rows <= a.least_rows || rows > a.most_rows) return h;
    h.tiles = (uint32_t)(rows + ROWS - 1) / ROWS;
    const int64_t seen = min((int64_t)held, (int64_t)a.window + ROWS / a.group + KEYS);
    h.units = max(1u, (uint32_t)((seen + KEYS - 1) / KEYS));
    return h;
}

template <class T>
__device__ __forceinline__ T wave_add(T v) {
#pragma unroll
    for (int off = kWave / 2; off > 0; off >>= 1) v += __shfl_xor(v, off, kWave);
    return v;
}

struct Item {
    Run run;
    int seq, length, tile, split, splits;
    int64_t slot;                                              // of its first split, among those of tiles that are cut
};

// The index-th part (CUT: the index-th tile that is cut) of the batch, in the order sequence, tile, split, the tiles with most keys first.  Tiles are cut so
// that a split has at least 1 / target of all the work: no more than `target` splits begin anew, whatever the lengths are, so that grids
// and workspaces are known on the host.
template <int ROWS, int KEYS, bool CUT>
__device__ bool find(const Attend &a, uint32_t index, uint32_t target, Item &it) {
    const int lane = threadIdx.x % kWave;
    Share mine = share_of<ROWS, KEYS>(a, lane);
    int64_t work = (int64_t)mine.tiles * mine.units;
    uint32_t most = mine.units;
    for (int s0 = kWave; s0 < a.p.seqs; s0 += kWave) {
        const Share h = share_of<ROWS, KEYS>(a, s0 + lane);
        work += (int64_t)h.tiles * h.units;
        most = max(most, h.units);
    }
    const int64_t per64 = (wave_add(work) * a.p.kv_heads + target - 1) / target;
    const int longest = __any(most > kSingle) ? kSingle + 1 : __any(most > kWhole) ? kSingle : kWhole;           // (as far as it matters)
    const int least = KEYS != kFewKeys * kFewWaves ? 1 : a.p.reach <= kUncut * KEYS ? kUncut : longest > kWhole && longest <= kSingle ? 1 : 2;
    const uint32_t per = (uint32_t)min(max(per64, (int64_t)least), (int64_t)INT32_MAX);
    uint32_t parts0 = 0;
    int64_t slots0 = 0;
    for (int s0 = 0; s0 < a.p.seqs; s0 += kWave) {
        if (s0) mine = share_of<ROWS, KEYS>(a, s0 + lane);
        mine.splits = (mine.units + per - 1) / per;
        const uint32_t all = mine.tiles * mine.splits;
        const uint32_t slots = mine.splits > 1 ? all : 0, parts = CUT ? (mine.splits > 1 ? mine.tiles : 0) : all;
        uint32_t sum_parts = parts, sum_slots = slots;
#pragma unroll
        for (int off = 1; off < kWave; off <<= 1) {
            const uint32_t u = __shfl_up(sum_parts, off, kWave), v = __shfl_up(sum_slots, off, kWave);
            if (lane >= off) { sum_parts += u; sum_slots += v; }
        }
        const uint32_t first = parts0 + sum_parts - parts;
        const uint64_t hit = __ballot(parts && index >= first && index - first < parts);
        if (hit) {
            const int from = __builtin_ctzll(hit);
            auto of = [&](uint32_t v) { return (uint32_t)__builtin_amdgcn_readlane((int)v, from); };
            const uint32_t rest = index - of(first), splits = of(mine.splits), tile = CUT ? rest : rest / splits;
            it.run = {(int)of(mine.run.first), (int)of(mine.run.n)};
            it.seq = s0 + from;
            it.length = (int)of(mine.length);
            it.splits = (int)splits;
            it.split = CUT ? 0 : (int)(rest - tile * splits);
            it.tile = (int)(of(mine.tiles) - 1 - tile);
            it.slot = slots0 + of(sum_slots - slots) + (int64_t)tile * splits;
            return true;
        }
        parts0 += __builtin_amdgcn_readlane((int)sum_parts, kWave - 1);
        slots0 += (uint32_t)__builtin_amdgcn_readlane((int)sum_slots, kWave - 1);
    }
    return false;
}

// Rows that belong to nobody, in front of the first sequence and behind the last, answer 0; the blocks of a launch share them.
__device__ void clear_rest(const Attend &a, int64_t block, int64_t blocks, int threads) {
    const int first = a.p.seqs ? min(max(a.p.offsets[0], 0), a.p.rows) : 0, used = a.p.seqs ? min(max(a.p.offsets[a.p.seqs], 0), a.p.rows) : 0;
    const int64_t row = (int64_t)a.heads * a.p.dim / 8, front = first * row, end = front + (a.p.rows - used) * row;
    for (int64_t i = block * threads + threadIdx.x; i < end; i += blocks * threads) reinterpret_cast<u32x4 *>(a.out)[i < front ? i : i - front + used * row] = u32x4{0, 0, 0, 0};
}

// ---------------------------------------------------------------------------------------------------------------- tiles in LDS
// A tile is [keys][D] bf16, its rows cut into pieces of 16 bytes that stand at piece ^ swizzle(row): for K so that the 16 rows that are read at a time,
// one piece each, lie in different banks; for V so that four rows, four pieces each, do.
template <int D>
__device__ __forceinline__ int swizzle_k(int row) { return D == 128 ? row & 15 : (row >> 1) & 7; }
template <int D>
__device__ __forceinline__ int swizzle_v(int row) { return D == 128 ? (row & 3) << 2 : ((row >> 1) & 1) << 2; }

// 16 bytes of each lane's to LDS at `to` + 16 * lane, without passing registers
__device__ __forceinline__ void to_lds(uint32_t to, const uint8_t *from) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(to), "v"(from) : "memory");
}
// and from an address of the wave's at a distance of the lane's
__device__ __forceinline__ void to_lds(uint32_t to, const uint8_t *from, uint32_t at) {
    const uint64_t v = reinterpret_cast<uint64_t>(from);       // (the same in all lanes, which the compiler does not always see)
    const uint64_t base = (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(v >> 32)) << 32 | (uint32_t)__builtin_amdgcn_readfirstlane((int)v);
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(to), "v"(at), "s"(base) : "memory");
}
// Everything asked for is in LDS, and everything read from there in registers: what is asked for next may take its place.
__device__ __forceinline__ void all_loads_done() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory"); }

__device__ __forceinline__ const uint8_t *shuffled(const uint8_t *p, int lane) {
    const uint64_t v = reinterpret_cast<uint64_t>(p);
    const uint32_t lo = __shfl((int)(uint32_t)v, lane, kWave), hi = __shfl((int)(uint32_t)(v >> 32), lane, kWave);
    return reinterpret_cast<const uint8_t *>((uint64_t)hi << 32 | lo);
}

// sixteen codes -> sixteen bf16 (exact: E4M3 has 3 bits of mantissa)
__device__ __forceinline__ void widen16(u32x4 codes, u32x4 &lo, u32x4 &hi) {
    uint32_t o[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const auto a = __builtin_amdgcn_cvt_pk_f32_fp8((int)codes[i], false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)codes[i], true);
        o[2 * i] = __builtin_amdgcn_perm(float_to_bits(a[1]), float_to_bits(a[0]), 0x07060302u);
        o[2 * i + 1] = __builtin_amdgcn_perm(float_to_bits(b[1]), float_to_bits(b[0]), 0x07060302u);
    }
    lo = u32x4{o[0], o[1], o[2], o[3]};
    hi = u32x4{o[4], o[5], o[6], o[7]};
}

// Where the token at a position lies; rows of zeros where there is none.
struct Place {
    const uint8_t *key, *value;
    bool held;
};
__device__ __forceinline__ Place place_of(const Paged &p, int page, int pos, int head) {
    const uint8_t *zeros = reinterpret_cast<const uint8_t *>(g_zeros);
    Place w = {zeros, zeros, page >= 0 && page < p.pages};
    if (w.held) {
        const int at = pos & ((1 << p.shift) - 1);
        w.key = p.keys + page * p.k_page + head * p.k_head + at * p.k_tok;
        w.value = p.values + page * p.v_page + head * p.v_head + at * p.v_tok;
    }
    return w;
}

// ---------------------------------------------------------------------------------------------------------------- the attention of 32 rows
// A block goes over its keys once; where the sums then say that there are infinities or NaN, which 0 * NaN may have brought to rows that do not see them,
// it goes over them again with zeros in their places, and once more to add them where they are seen.
enum Pass { kOnce, kFinite, kOdd };

// exchange with lane ^ 32
__device__ __forceinline__ float other_half(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(float_to_bits(v), float_to_bits(v), false, false);
    return bits_to_float(threadIdx.x % kWave < 32 ? r[1] : r[0]);
}

// A lane's 32 rows by 16 of 32 keys (element i is key 8 (i / 4) + 4 (lane / 32) + i % 4), NB such blocks of keys a tile.  C of the D
// columns that tiles have room for are multiplied.
template <int D, int NB, int C = D>
struct Rows32 {
    bf16x8 q[C / 16];
    f32x16 o[C / 32];
    f32x16 s[NB];                                              // of a tile: scores, weights as fp32
    bf16x8 w[2 * NB];                                          // and as bf16
    float m, l;                                                // running maximum in powers of two, the sum of this lane's keys against it

    __device__ __forceinline__ void start() {
        m = -INFINITY;
        l = 0.0f;
#pragma unroll
        for (int d = 0; d < C / 32; ++d) o[d] = f32x16{};
    }

    // Rows first_row + lane % 32 of a tile's: q of a token's head, zeros where there is no such row; the other sign where `negative` (see caps_of).  Every lane reads, those without a
    // row the sequence's first token and pieces behind head_dim the first one: around masked loads the compiler may spill what all lanes need, for the lanes that are on
    // alone.  (One token behind 200, heads of 128: 0.3 of 10 us.)
    __device__ __forceinline__ void load_q(const Attend &a, const Run &run, int row, int kv_head, bool negative) {
        const int lane = threadIdx.x % kWave, token = row / a.group, head = kv_head * a.group + row % a.group;
        const bool live = token < run.n;
        const uint16_t *from = a.q + (int64_t)(run.first + (live ? token : 0)) * a.q_row + head * a.q_head;
        const uint32_t sign = negative ? 0x80008000u : 0u;
#pragma unroll
        for (int s = 0; s < C / 16; ++s) {
            const int c = 16 * s + 8 * (lane / 32);
            u32x4 v = *reinterpret_cast<const u32x4 *>(from + (c < a.p.dim ? c : 0));
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = live && c < a.p.dim ? v[i] ^ sign : 0u;
            q[s] = __builtin_bit_cast(bf16x8, v);
        }
    }

    // One tile in three steps.  Scores of the keys at LDS address kt:
    __device__ __forceinline__ void scores(uint32_t kt) {
        const int lane = threadIdx.x % kWave, h = lane / 32, r = lane % 32;
        const uint32_t at = kt + r * 2 * D + 16 * (h ^ swizzle_k<D>(r));
#pragma unroll
        for (int b = 0; b < NB; ++b) s[b] = f32x16{};
#pragma unroll
        for (int d = 0; d < C / 16; ++d) {
            const lds_u8 *from = (const lds_u8 *)(uintptr_t)(at ^ (32 * d));
#pragma unroll
            for (int b = 0; b < NB; ++b)
                s[b] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(*(const __attribute__((address_space(3))) bf16x8 *)(from + b * 32 * 2 * D), q[d], s[b], 0, 0, 0);
        }
    }

    // Scores capped, and then in powers of two: out * tanh(x), in * s = 2 x log2 e.  1 - 2 / (e^2x + 1) is off by up to 5 * 2^-24, and a score by as much of the cap: up to a cap
    // of 256 that is 8e-5, a fiftieth of what a weight's rounding to bf16 is.  With larger caps scores are off by some 2^-24 of themselves: up to 1/2, tanh(x) = x p(x^2), p fitted to
    // relative 2^-25, and only from there on the quotient, where the 1 costs no more than a digit.  (With that for every cap the chunk above, capped at 30, takes 708 us, 1300 where
    // scores are large, and not 670.)
    __device__ __forceinline__ void cap(float in, float out) {
        auto far = [&](float v) { return __fmaf_rn(-2.0f * out, __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(v * in) + 1.0f), out); };
        auto all = [&](auto f) {
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int i = 0; i < 16; ++i) s[b][i] = f(s[b][i]);
        };
        if (out <= 256.0f * kLog2e) return all(far);
        float by = in;
        asm volatile("" : "+v"(by));             // (so that nothing of what follows is kept in registers for it)
        by *= 0.5f / kLog2e;
        auto near = [&](float v) {
            const float x = v * by, y = x * x;
            return out * (x * __fmaf_rn(__fmaf_rn(__fmaf_rn(__fmaf_rn(1.72414854e-2f, y, -5.30454926e-2f), y, 1.3325879e-1f), y, -3.33331436e-1f), y, 1.0f));
        };
        float most = 0.0f;
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int i = 0; i < 16; ++i) most = fmaxf(most, __builtin_fabsf(s[b][i]));
        if (!__any(most * by > 0.5f)) return all(near);
        all([&](float v) { return __builtin_fabsf(v * by) > 0.5f ? far(v) : near(v); });
    }

    // Scores of keys that the lane's row does not see go: of seen, bit e is key e + 4 (lane / 32), for e % 8 < 4.
    __device__ __forceinline__ void hide(uint64_t seen) {
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int i = 0; i < 16; ++i) s[b][i] = (uint32_t)(seen >> 32 * b) & 1u << (8 * (i / 4) + i % 4) ? s[b][i] : -INFINITY;
    }

    // Weights from scores.  c: powers of two a unit of a score.
    __device__ __forceinline__ void weights(float c) {
        float top = -INFINITY;
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int i = 0; i < 16; ++i) top = fmaxf(top, s[b][i]);
        top = fmaxf(top, other_half(top)) * c;
        // The maximum may lag by 2^8: weights are then up to 2^8, in types that hold that as well, and most tiles leave sums as they are.
        if (__any(top > m + kSlack)) {
            const float to = fmaxf(m, top), by = to == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - to);
            m = to;
            l *= by;
#pragma unroll
            for (int d = 0; d < C / 32; ++d)
#pragma unroll
                for (int i = 0; i < 16; ++i) o[d][i] *= by;
        }
        const float against = m == -INFINITY ? 0.0f : m;
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                s[b][i] = __builtin_amdgcn_exp2f(__fmaf_rn(s[b][i], c, -against));
                l += s[b][i];
            }
#pragma unroll
        for (int k = 0; k < 2 * NB; ++k) {
            uint32_t v[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = pack_bf16x2(s[k / 2][8 * (k % 2) + 2 * i], s[k / 2][8 * (k % 2) + 2 * i + 1]);
            u32x4 packed = {v[0], v[1], v[2], v[3]};
            asm volatile("" : "+v"(packed));                   // (here, and not where they are used first: that is the other half's turn)
            w[k] = __builtin_bit_cast(bf16x8, packed);
        }
    }

    // The weighted values at LDS address vt.
    __device__ __forceinline__ void sums(uint32_t vt) {
        const uint32_t at = value_address(vt);
#pragma unroll
        for (int k = 0; k < 2 * NB; ++k)
#pragma unroll
            for (int d = 0; d < C / 32; ++d)
                o[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, values(at, d, k)), w[k], o[d], 0, 0, 0);
    }

    // The weighted values of one tile and the scores of another, both steps' operands four at a time and a group ahead (left to itself the compiler reads each
    // where it is used, and waits: 2350 cycles, of which 1024 multiply; two groups ahead keep 16 registers more in scratch memory: a chunk of 2048 tokens behind
    // 14336 takes 526 us and not 500).
    __device__ __forceinline__ void sums_and_scores(uint32_t vt, uint32_t kt) {
        constexpr int kColumns = C / 32, kSums = 2 * NB * kColumns, kGroups = (kSums + C / 16 * NB) / 4, kAhead = 1;
        static_assert(kSums % 4 == 0 && C / 16 * NB % 4 == 0, "groups");
        const int lane = threadIdx.x % kWave, h = lane / 32, r = lane % 32;
        const uint32_t v_at = value_address(vt), k_at = kt + r * 2 * D + 16 * (h ^ swizzle_k<D>(r));
        u32x4 f[kAhead + 1][4];
        auto read = [&](int g) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int n = 4 * g + i, m = n - kSums;
                f[g % (kAhead + 1)][i] = n < kSums ? values(v_at, n % kColumns, n / kColumns)
                                                   : *(const __attribute__((address_space(3))) u32x4 *)(uintptr_t)((k_at ^ (32 * (m / NB))) + m % NB * 32 * 2 * D);
            }
        };
        auto multiply = [&](int g) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int n = 4 * g + i, m = n - kSums;
                const bf16x8 x = __builtin_bit_cast(bf16x8, f[g % (kAhead + 1)][i]);
                if (n < kSums) o[n % kColumns] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(x, w[n / kColumns], o[n % kColumns], 0, 0, 0);
                else s[m % NB] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(x, q[m / NB], m < NB ? f32x16{} : s[m % NB], 0, 0, 0);
            }
        };
#pragma unroll
        for (int g = 0; g < kAhead; ++g) read(g);
#pragma unroll
        for (int g = 0; g < kGroups; ++g) {
            if (g + kAhead < kGroups) read(g + kAhead);
            __builtin_amdgcn_sched_barrier(0);
            multiply(g);
            __builtin_amdgcn_sched_barrier(0);
        }
    }

    // Lane i of 16 reads 4 of 16 columns of key i / 4, and gets 4 keys of column i.
    static __device__ __forceinline__ uint32_t value_address(uint32_t vt) {
        const int lane = threadIdx.x % kWave, i = lane % 16, key = 4 * (lane / 32) + i / 4;
        const int piece = (2 * ((lane / 16) % 2) + (i % 4) / 2) ^ swizzle_v<D>(key);
        return vt + key * 2 * D + piece * 16 + (i % 2) * 8;
    }
    // V^T of columns 32 d to 32 d + 31, keys 16 k + {0 to 3, 8 to 11} + 4 (lane / 32)
    static __device__ __forceinline__ u32x4 values(uint32_t at, int d, int k) {
        const uint32_t from = (at ^ (64 * d)) + k * 16 * 2 * D;
        const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4 *)(uintptr_t)from);
        const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4 *)(uintptr_t)(from + 8 * 2 * D));
        const u32x2 a = __builtin_bit_cast(u32x2, lo), b = __builtin_bit_cast(u32x2, hi);
        return u32x4{a[0], a[1], b[0], b[1]};
    }

    // Infinities and NaN among a tile's values, for the rows that see them (bit k: key k): weights are above 0, so they come through as they are.
    __device__ __forceinline__ void add_odd(uint32_t vt, uint64_t seen) {
        const int h = threadIdx.x % kWave / 32;
#pragma unroll 1
        for (int key = 0; key < 32 * NB; ++key) {
#pragma unroll
            for (int d = 0; d < C / 32; ++d)
#pragma unroll
                for (int i = 0; i < 4; ++i) {    // columns 32 d + 8 i + 4 h to + 3
                    const u32x2 v = *(const __attribute__((address_space(3))) u32x2 *)(uintptr_t)(vt + key * 2 * D + 16 * ((4 * d + i) ^ swizzle_v<D>(key)) + 8 * h);
#pragma unroll
                    for (int z = 0; z < 4; ++z) {
                        const float f = z % 2 ? bf16_hi(v[z / 2]) : bf16_lo(v[z / 2]);
                        if ((seen >> key & 1) && !(__builtin_fabsf(f) < INFINITY)) o[d][4 * i + z] += f;
                    }
                }
        }
    }

    // Whether a sum of this lane's rows is not finite.
    __device__ __forceinline__ bool odd() const {
        float most = 0.0f;
#pragma unroll
        for (int d = 0; d < C / 32; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i) most = fmaxf(most, o[d][i] != o[d][i] ? INFINITY : __builtin_fabsf(o[d][i]));
        return !(most < INFINITY);
    }
};

// Which keys of the tile from `base` on a row at position pos sees.  held: which there are.
__device__ __forceinline__ uint64_t seen_of(int pos, int base, int window, uint64_t held) {
    const int last = pos - base;
    const int64_t first = (int64_t)last - window + 1;
    uint64_t seen = last < 0 ? 0 : last >= 63 ? ~0ull : (2ull << last) - 1;
    if (first > 0) seen = first > 63 ? 0 : seen & (~0ull << first);
    return seen & held;
}

// The keys that a tile of rows sees, in units of KEYS: from `first` (aligned) to `end`.
struct Range {
    int first, end;
};
template <int ROWS, int KEYS>
__device__ __forceinline__ Range range_of(const Attend &a, const Item &it) {
    const int tokens = it.run.n, t0 = it.tile * ROWS / a.group, t1 = min((it.tile * ROWS + ROWS - 1) / a.group, tokens - 1);
    const int pos0 = it.length - tokens + t0, pos1 = it.length - tokens + t1;
    const int held = min(max(it.length, 0), a.p.reach);
    const int64_t from = (int64_t)pos0 - a.window + 1;
    Range r;
    r.first = from > 0 ? (int)(from / KEYS * KEYS) : 0;
    r.end = min(held, pos1 + 1);
    const int units = max(0, (r.end - r.first + KEYS - 1) / KEYS), each = (units + it.splits - 1) / it.splits;
    const int first = r.first + min(it.split * each, units) * KEYS;
    r.end = min(r.end, r.first + min((it.split + 1) * each, units) * KEYS);
    r.first = first;
    return r;
}

__device__ __forceinline__ void store_row(const Attend &a, const Run &run, int row, int kv_head, int d, f32x4 v) {
    const int token = row / a.group, head = kv_head * a.group + row % a.group;
    *reinterpret_cast<u32x2 *>(a.out + ((int64_t)(run.first + token) * a.heads + head) * a.p.dim + d) = u32x2{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])};
}

// What a sum against maximum m counts where `top` is the maximum of all.  A part that sees nothing has maximum -inf and sums 0, one that sees only NaN
// -inf and NaN.  No part counts nothing: an infinity that a row sees is its answer whatever its part weighs, and 2^-149 of any finite sum is none to be seen.
__device__ __forceinline__ float weight_of(float m, float top) { return m == top ? 1.0f : fmaxf(__builtin_amdgcn_exp2f(m - top), __FLT_DENORM_MIN__); }
// A row's answer from its sums; a row that sees nothing, or no score above -inf, answers 0, infinities and NaN among its values or not.
__device__ __forceinline__ float quotient_of(const Attend &a, int kv_head, float l) { return (a.p.value_scale ? a.p.value_scale[kv_head] : 1.0f) / l; }
__device__ __forceinline__ f32x4 answer_of(f32x4 o, float l, float quotient) { return l == 0.0f ? f32x4{0.0f, 0.0f, 0.0f, 0.0f} : o * quotient; }

// Scores from products: c powers of two a unit, or a cap's in and out.  A sign of the keys' scale goes into q, so that larger products are larger scores; with a scale of 0 all
// scores are 0, which the least c above 0 makes of them too, and hidden ones stay -inf.
struct Caps {
    float c, in, out;
    bool negative;
};
template <bool CAP>
__device__ __forceinline__ Caps caps_of(const Attend &a, int kv_head) {
    auto one = [](float v) { return bits_to_float((uint32_t)__builtin_amdgcn_readfirstlane((int)float_to_bits(v))); };       // (the same in all lanes: a scalar register)
    const float of_keys = a.p.key_scale ? a.p.key_scale[kv_head] : 1.0f, scale = a.scale * __builtin_fabsf(of_keys);
    if (CAP) return {1.0f, one(2.0f * kLog2e * scale / a.softcap), one(a.softcap * kLog2e), of_keys < 0.0f};
    const float c = scale * kLog2e;
    return {one(c == 0.0f ? __FLT_DENORM_MIN__ : c), 0.0f, 0.0f, of_keys < 0.0f};
}

// ---------------------------------------------------------------------------------------------------------------- keys and values on their way to LDS
// A wave's KEYS rows of a tile of keys or values, `first` to first + KEYS, from their places (lane i has that of the tile's row i) to LDS at `tile`.
// bf16 goes there directly; codes pass registers, where they are widened.
template <int D, int KEYS, bool E4M3, bool VALUES>
struct Stager;

template <int D, bool VALUES>
__device__ __forceinline__ int swizzle(int row) { return VALUES ? swizzle_v<D>(row) : swizzle_k<D>(row); }

template <int D, int KEYS, bool VALUES>
struct Stager<D, KEYS, false, VALUES> {
    static constexpr int kPieces = D / 8, kEach = kWave / kPieces, kLoads = KEYS / kEach;      // pieces of a row, rows a load
    __device__ __forceinline__ void fetch(const uint8_t *place, int first, int dim, uint32_t tile) const {
        const int lane = threadIdx.x % kWave, piece = lane % kPieces;
        const uint8_t *zeros = reinterpret_cast<const uint8_t *>(g_zeros);
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            const int row = first + i * kEach + lane / kPieces, c = piece ^ swizzle<D, VALUES>(row);
            const uint8_t *from = shuffled(place, row);
            to_lds(tile + (first + i * kEach) * 2 * D, (c * 8 < dim ? from : zeros) + c * 16);
        }
    }
    // the i-th load from one page
    __device__ __forceinline__ void one(int i, const uint8_t *page, uint32_t at, bool in, int first, uint32_t tile) const {
        if (in) to_lds(tile + (first + i * kEach) * 2 * D, page, at);
    }
    __device__ __forceinline__ void put(int, uint32_t) const { all_loads_done(); }
};

template <int D, int KEYS, bool VALUES>
struct Stager<D, KEYS, true, VALUES> {
    static constexpr int kPieces = D / 16, kEach = kWave / kPieces < KEYS ? kWave / kPieces : KEYS, kLoads = KEYS / kEach;
    u32x4 codes[kLoads];
    __device__ __forceinline__ void fetch(const uint8_t *place, int first, int dim, uint32_t) {
        const int lane = threadIdx.x % kWave, piece = lane % kPieces;
        const uint8_t *zeros = reinterpret_cast<const uint8_t *>(g_zeros);
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            const uint8_t *from = shuffled(place, first + i * kEach + lane / kPieces % kEach);
            codes[i] = *reinterpret_cast<const u32x4 *>((piece * 16 < dim ? from : zeros) + piece * 16);
        }
    }
    __device__ __forceinline__ void one(int i, const uint8_t *page, uint32_t at, bool in, int, uint32_t) {
        codes[i] = u32x4{0, 0, 0, 0};
        if (in) codes[i] = *reinterpret_cast<const u32x4 *>(page + at);
    }
    __device__ __forceinline__ void put(int first, uint32_t tile) const {
        const int lane = threadIdx.x % kWave, piece = lane % kPieces;
        if (lane / kPieces >= kEach) return;
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            const int row = first + i * kEach + lane / kPieces, z = swizzle<D, VALUES>(row);
            u32x4 lo, hi;
            widen16(codes[i], lo, hi);
            *(__attribute__((address_space(3))) u32x4 *)(uintptr_t)(tile + row * 2 * D + 16 * ((2 * piece) ^ z)) = lo;
            *(__attribute__((address_space(3))) u32x4 *)(uintptr_t)(tile + row * 2 * D + 16 * ((2 * piece + 1) ^ z)) = hi;
        }
    }
};

// Zeros in the place of infinities and NaN, in 16-byte pieces first, first + step, .. of a tile of values.
__device__ __forceinline__ void make_finite(uint32_t vt, int first, int step, int pieces) {
#pragma unroll 1
    for (int i = first; i < pieces; i += step) {
        auto at = (__attribute__((address_space(3))) u32x4 *)(uintptr_t)(vt + 16 * i);
        u32x4 v = *at;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if ((v[k] & 0x7f80u) == 0x7f80u) v[k] &= 0xffff0000u;
            if ((v[k] & 0x7f800000u) == 0x7f800000u) v[k] &= 0xffffu;
        }
        *at = v;
    }
}

__device__ __forceinline__ uint32_t lds_base(uint8_t *lds) { return (uint32_t)(uintptr_t)(lds_u8 *)lds; }

// ---------------------------------------------------------------------------------------------------------------- few rows
template <int D, bool E4M3, bool CAP>
__global__ __launch_bounds__(kFewWaves *kWave, E4M3 ? 2 : 1) void attend_few_kernel(Attend a) {
    extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
    constexpr int kTile = kFewKeys * 2 * D, kStages = E4M3 ? 1 : 2, kStep = kFewKeys * kFewWaves;
    const int head = blockIdx.x % a.p.kv_heads, lane = threadIdx.x % kWave;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    clear_rest(a, blockIdx.x, gridDim.x, kFewWaves * kWave);
    Item it;
    if (!find<kFewRows, kStep, false>(a, blockIdx.x / a.p.kv_heads, few_target(D, E4M3), it)) return;
    const Range range = range_of<kFewRows, kStep>(a, it);
    const int rows = it.run.n * a.group, row0 = it.tile * kFewRows, row = row0 + lane % 32, before = it.length - it.run.n;
    const int pos = before + row / a.group, pos0 = before + row0 / a.group, pos1 = before + min(row0 + kFewRows - 1, rows - 1) / a.group;
    const Caps caps = caps_of<CAP>(a, head);
    const int32_t *table = a.p.table + it.seq * a.p.table_stride;
    Rows32<D, 1> w;
    w.load_q(a, it.run, row, head, E4M3 && caps.negative);

    const int h4 = 4 * (lane / 32);
    Pass pass = kOnce;
    const uint32_t mine = lds_base(lds) + wave * kStages * 2 * kTile;
    auto page_of = [&](int base) { return base + lane % 32 < range.end ? table[(base + lane % 32) >> a.p.shift] : -1; };
    auto attend = [&](int base, uint32_t held, uint32_t kt) {
        const uint64_t seen = seen_of(pos, base, a.window, held);
        if (pass == kOdd) {
            w.add_odd(kt + kTile, seen);
            return;
        }
        if (pass == kFinite) make_finite(kt + kTile, lane, kWave, kTile / 16);
        w.scores(kt);
        if (CAP) w.cap(caps.in, caps.out);
        if (held != ~0u || base + kFewKeys - 1 > pos0 || base <= pos1 - a.window) w.hide(seen >> h4);
        w.weights(caps.c);
        w.sums(kt + kTile);
    };
    for (;;) {
        if (pass != kOdd) w.start();
        int base = range.first + wave * kFewKeys;
        int page = page_of(base);
        uint32_t held = 0, stage = 0;
        Stager<D, kFewKeys, E4M3, false> keys;
        Stager<D, kFewKeys, E4M3, true> values;
        auto fetch = [&](int at) {               // the tile at `at`, whose pages are known; then the pages of the next
            const Place place = place_of(a.p, page, at + lane % 32, head);
            held = (uint32_t)__ballot(place.held);
            keys.fetch(place.key, 0, a.p.dim, mine + stage);
            values.fetch(place.value, 0, a.p.dim, mine + stage + kTile);
            page = page_of(at + kStep);
        };
        if (base < range.end) fetch(base);
        for (; base < range.end; base += kStep) {
            const uint32_t now = held, kt = mine + stage;
            keys.put(0, kt);
            values.put(0, kt + kTile);
            if (!E4M3) stage ^= 2 * kTile;
            if (base + kStep < range.end) fetch(base + kStep);
            attend(base, now, kt);
        }
        if (pass == kOdd || (pass == kOnce && !__any(w.odd()))) break;
        pass = pass == kOnce ? kFinite : kOdd;
    }
    w.l += other_half(w.l);

    // the four waves' sums as one
    __syncthreads();
    constexpr int kRow = D + 4;                  // floats: rows begin in other banks
    float *sums = reinterpret_cast<float *>(lds), *ml = sums + kFewWaves * 32 * kRow;
    const int r = lane % 32, used = min(rows - row0, 32);
    if (lane < 32) {
        ml[(wave * 32 + r) * 2] = w.m;
        ml[(wave * 32 + r) * 2 + 1] = w.l;
    }
    __syncthreads();
    float top = ml[r * 2];
#pragma unroll
    for (int v = 1; v < kFewWaves; ++v) top = fmaxf(top, ml[(v * 32 + r) * 2]);
    const float part = weight_of(w.m, top);
    if (r < used) {
#pragma unroll
        for (int d = 0; d < D / 32; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                *reinterpret_cast<f32x4 *>(sums + (wave * 32 + r) * kRow + 32 * d + 8 * i + 4 * (lane / 32)) =
                    f32x4{w.o[d][4 * i] * part, w.o[d][4 * i + 1] * part, w.o[d][4 * i + 2] * part, w.o[d][4 * i + 3] * part};
    }
    __syncthreads();
    const int64_t slot = (it.slot + it.split) * a.p.kv_heads + head;
    for (int e = threadIdx.x; e < used * (D / 4); e += kFewWaves * kWave) {
        const int rr = e / (D / 4), d = e % (D / 4) * 4;
        float m = ml[rr * 2];
#pragma unroll
        for (int v = 1; v < kFewWaves; ++v) m = fmaxf(m, ml[(v * 32 + rr) * 2]);
        f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
        float l = 0.0f;
#pragma unroll
        for (int v = 0; v < kFewWaves; ++v) {
            o += *reinterpret_cast<const f32x4 *>(sums + (v * 32 + rr) * kRow + d);
            l = __fmaf_rn(ml[(v * 32 + rr) * 2 + 1], weight_of(ml[(v * 32 + rr) * 2], m), l);
        }
        if (it.splits == 1) {
            if (d < a.p.dim) store_row(a, it.run, row0 + rr, head, d, answer_of(o, l, quotient_of(a, head, l)));
        } else if (slot < a.slots) {
            *reinterpret_cast<f32x4 *>(a.partial + (slot * kFewRows + rr) * D + d) = o;
            if (d == 0) {
                float *to = a.partial + a.slots * kFewRows * D + (slot * kFewRows + rr) * 2;
                to[0] = m;
                to[1] = l;
            }
        }
    }
}

// ---------------------------------------------------------------------------------------------------------------- many rows
// Whether a wave is the second (fourth, ..) of its block on its SIMD.  lds: room for a number of each wave, which nothing else uses yet.
template <int WAVES>
__device__ __forceinline__ bool second_of_simd(uint8_t *lds, int wave) {
    constexpr int kHwId = 4, kOffset = 4, kBits = 2;           // of the register that says where a wave runs, its SIMD
    const int simd = __builtin_amdgcn_s_getreg(kHwId | kOffset << 6 | (kBits - 1) << 11);
    int *at = reinterpret_cast<int *>(lds);
    if (threadIdx.x % kWave == 0) at[wave] = simd;
    __syncthreads();
    int before = 0;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) before += w < wave && at[w] == simd;
    __syncthreads();
    return __builtin_amdgcn_readfirstlane(before & 1);
}

// The eight waves in two halves, each with a wave on every SIMD: while one half multiplies, the other makes weights, and a barrier turns them.  In the
// half's turn at the matrix units a wave adds up the values of tile t - 1 and makes the scores of tile t.
//   step          0        1        2        3        4
//   first half    s0       w0       o0 s1    w1       o1 s2    ..         K(t) and V(t - 1) are read in steps 2 t and 2 t + 1; three tiles of each are in
//   second half            s0       w0       o0 s1    w1       ..         LDS, so that those of t + 2 can be asked for while the half makes weights of t
constexpr int many_lds(int D) { return 3 * 2 * kManyKeys * 2 * D; }

// A wave's eight rows of a tile in one page: one address for the wave and each lane's distance from it, worked out once.  Pieces behind head_dim are
// neither read nor written.
template <int D, bool E4M3>
struct Eight {
    static constexpr int kPieces = E4M3 ? D / 16 : D / 8, kEach = kWave / kPieces < 8 ? kWave / kPieces : 8, kLoads = 8 / kEach;
    uint32_t k_at[kLoads], v_at[kLoads];
    bool k_in[kLoads], v_in[kLoads], paged;
    __device__ __forceinline__ void start(const Paged &p, int first) {
        const int lane = threadIdx.x % kWave, piece = lane % kPieces;
        paged = p.shift >= 3 && p.k_tok < 1 << 24 && p.v_tok < 1 << 24;
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            const int r = i * kEach + lane / kPieces;
            const int ck = E4M3 ? piece : piece ^ swizzle_k<D>(first + r), cv = E4M3 ? piece : piece ^ swizzle_v<D>(first + r);
            k_at[i] = r * (uint32_t)p.k_tok + ck * 16;
            v_at[i] = r * (uint32_t)p.v_tok + cv * 16;
            k_in[i] = ck * (E4M3 ? 16 : 8) < p.dim && r < 8;
            v_in[i] = cv * (E4M3 ? 16 : 8) < p.dim && r < 8;
        }
    }
};

template <int D, int C, bool E4M3, bool CAP>
__global__ __launch_bounds__(kManyWaves *kWave) void attend_many_kernel(Attend a, int clear) {
    extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
    constexpr int kTile = kManyKeys * 2 * D, kMine = kManyKeys / kManyWaves;
    const int head = blockIdx.x % a.p.kv_heads, lane = threadIdx.x % kWave;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const bool second = second_of_simd<kManyWaves>(lds, wave);
    if (clear) clear_rest(a, blockIdx.x, gridDim.x, kManyWaves * kWave);
    Item it;
    if (!find<kManyRows, kManyKeys, false>(a, blockIdx.x / a.p.kv_heads, kManyTarget, it)) return;
    const Range range = range_of<kManyRows, kManyKeys>(a, it);
    const int rows = it.run.n * a.group, row0 = it.tile * kManyRows + 32 * wave, row = row0 + lane % 32, before = it.length - it.run.n;
    const int pos = before + row / a.group, pos0 = before + row0 / a.group, pos1 = before + min(row0 + 31, rows - 1) / a.group;
    const Caps caps = caps_of<CAP>(a, head);
    const int32_t *table = a.p.table + it.seq * a.p.table_stride;
    const int tiles = (range.end - range.first + kManyKeys - 1) / kManyKeys;
    Rows32<D, 2, C> w;
    w.load_q(a, it.run, row, head, E4M3 && caps.negative);

    const uint32_t keys = lds_base(lds), values = keys + 3 * kTile;
    const int h4 = 4 * (lane / 32);
    bool finite = false;
    Stager<D, kMine, E4M3, false> key_stager;
    Stager<D, kMine, E4M3, true> value_stager;
    const int mine = wave * kMine;
    static_assert(kMine == 8, "rows of a wave");
    Eight<D, E4M3> eight;
    eight.start(a.p, mine);
    if (!E4M3 && a.p.dim < D) {                  // (what no load writes)
        for (int i = threadIdx.x; i < many_lds(D) / 16; i += kManyWaves * kWave) reinterpret_cast<u32x4 *>(lds)[i] = u32x4{0, 0, 0, 0};
        __syncthreads();
    }
    auto base_of = [&](int t) { return range.first + t * kManyKeys; };
    auto page_of = [&](int t) { return base_of(t) + lane < range.end ? table[(base_of(t) + lane) >> a.p.shift] : -1; };
    // Where this wave's rows of 64 tiles to come lie, a lane a tile (0: every lane has its own place), and which keys of the tile there are.
    using E = Eight<D, E4M3>;
    uint64_t key_of = 0, value_of = 0, held_of = 0;
    auto look_ahead = [&](int t0) {
        const int base = base_of(t0 + lane);
        uint64_t keys_held = 0;
        int id = -1;
#pragma unroll
        for (int g = 0; g < kManyWaves; ++g) {
            const int pos = base + 8 * g, page = pos < range.end ? table[pos >> a.p.shift] : -1;
            if ((uint32_t)page < (uint32_t)a.p.pages) keys_held |= 0xffull << 8 * g;
            if (g == wave) id = page;
        }
        const int pos = base + mine, at = pos & ((1 << a.p.shift) - 1), left = range.end - base;
        held_of = left >= kManyKeys ? keys_held : left <= 0 ? 0 : keys_held & ~(~0ull << left);
        const bool together = eight.paged && pos + kMine <= range.end && (uint32_t)id < (uint32_t)a.p.pages;
        key_of = together ? reinterpret_cast<uint64_t>(a.p.keys + id * a.p.k_page + head * a.p.k_head + at * a.p.k_tok) : 0;
        value_of = together ? reinterpret_cast<uint64_t>(a.p.values + id * a.p.v_page + head * a.p.v_head + at * a.p.v_tok) : 0;
    };
    auto of_lane = [](uint64_t v, int lane) {
        return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), lane) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)v, lane);
    };
    struct Where {
        const uint8_t *at;                       // the wave's first row, null where every lane has its own place
        const uint8_t *place;
    } key = {a.p.keys, a.p.keys}, value = {a.p.values, a.p.values};
    uint64_t held[2];                            // of the last tile asked for and of the one in front of it (1, 0)
    const bool whole = a.p.dim == D && E::kEach * E::kPieces == kWave;
    auto fetch = [&](int t, uint32_t kt, uint32_t vt) {        // keys of tile t, values of the one in front of it
        if (t % kWave == 0) look_ahead(t);
        held[0] = held[1];
        held[1] = of_lane(held_of, t % kWave);
        if (t > 0 && t <= tiles) {
            if (value.at) {
#pragma unroll
                for (int i = 0; i < E::kLoads; ++i) value_stager.one(i, value.at, eight.v_at[i], whole || eight.v_in[i], mine, vt);
            } else {
                value_stager.fetch(value.place, mine, a.p.dim, vt);
            }
        }
        if (t >= tiles) return;
        key.at = reinterpret_cast<const uint8_t *>(of_lane(key_of, t % kWave));
        value.at = reinterpret_cast<const uint8_t *>(of_lane(value_of, t % kWave));
        if (key.at) {
#pragma unroll
            for (int i = 0; i < E::kLoads; ++i) key_stager.one(i, key.at, eight.k_at[i], whole || eight.k_in[i], mine, kt);
        } else {
            const int at = base_of(t) + lane;
            const Place place = place_of(a.p, at < range.end ? table[at >> a.p.shift] : -1, at, head);
            held[1] = __ballot(place.held);
            key_stager.fetch(place.key, mine, a.p.dim, kt);
            value.place = place.value;
        }
    };
    auto arrived = [&](int t, uint32_t kt, uint32_t vt) {
        if (t < tiles) key_stager.put(mine, kt);
        if (t > 0 && t <= tiles) {
            value_stager.put(mine, vt);
            if (finite) make_finite(vt + mine * 2 * D, lane, kWave, kMine * 2 * D / 16);
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    };
    auto turn = [&]() {
        __builtin_amdgcn_sched_barrier(0);
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_sched_barrier(0);
        asm volatile("" ::: "memory");
    };
    for (;;) {
        w.start();
        uint32_t b0 = 0, b1 = kTile, b2 = 2 * kTile;           // where tiles t, t + 1 and t + 2 lie
        fetch(0, keys + b0, 0);
        arrived(0, keys + b0, 0);
        fetch(1, keys + b1, values + b0);
        turn();
        if (second) turn();
        w.scores(keys + b0);
        arrived(1, keys + b1, values + b0);
        turn();
        for (int t = 0; t < tiles; ++t) {
            const int base = base_of(t);
            if (CAP) w.cap(caps.in, caps.out);
            if (held[0] != ~0ull || base + kManyKeys - 1 > pos0 || base <= pos1 - a.window) w.hide(seen_of(pos, base, a.window, held[0]) >> h4);
            w.weights(caps.c);
            fetch(t + 2, keys + b2, values + b1);
            turn();
            w.sums_and_scores(values + b0, keys + b1);          // (scores behind the last tile: of what was there, for nobody)
            arrived(t + 2, keys + b2, values + b1);
            turn();
            const uint32_t b = b0;
            b0 = b1, b1 = b2, b2 = b;
        }
        if (!second) turn();
        if (!__syncthreads_or(w.odd()) || finite) break;
        finite = true;
    }
    if (finite)
        for (int t = 0; t < tiles; ++t) {
            const Place place = place_of(a.p, page_of(t), base_of(t) + lane, head);
            value_stager.fetch(place.value, mine, a.p.dim, values);
            value_stager.put(mine, values);
            __syncthreads();
            w.add_odd(values, seen_of(pos, base_of(t), a.window, __ballot(place.held)));
            __syncthreads();
        }
    w.l += other_half(w.l);
    if (row >= rows) return;
    const int64_t slot = (it.slot + it.split) * a.p.kv_heads + head;
    const float by = quotient_of(a, head, w.l);
#pragma unroll
    for (int d = 0; d < C / 32; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int at = 32 * d + 8 * i + 4 * (lane / 32);
            const f32x4 o = {w.o[d][4 * i], w.o[d][4 * i + 1], w.o[d][4 * i + 2], w.o[d][4 * i + 3]};
            if (it.splits == 1) {
                if (at < a.p.dim) store_row(a, it.run, row, head, at, answer_of(o, w.l, by));
            } else if (slot < a.slots) {
                *reinterpret_cast<f32x4 *>(a.partial + (slot * kManyRows + row - it.tile * kManyRows) * D + at) = o;
            }
        }
    if (it.splits > 1 && slot < a.slots && lane < 32) {
        float *to = a.partial + a.slots * kManyRows * D + (slot * kManyRows + row - it.tile * kManyRows) * 2;
        to[0] = w.m;
        to[1] = w.l;
    }
}

// ---------------------------------------------------------------------------------------------------------------- splits as one
// A block has some rows of a tile that was cut.  First the weights of their splits, a lane a row and split, then the sums: the block's lanes in groups that
// share the splits, each in order, and are added up in order.
constexpr int kJoinFew = 4, kJoinMany = 32;                   // rows of a block

template <int D, int ROWS, int KEYS, int MINE>
__global__ __launch_bounds__(256) void attend_join_kernel(Attend a, uint32_t target) {
    constexpr int kColumns = D / 4, kItems = MINE * kColumns, kGroups = kItems < 256 ? 256 / kItems : 1, kSplits = 2048 / MINE;
    __shared__ float weight[MINE][kSplits], tops[MINE], totals[MINE];
    __shared__ f32x4 part[kGroups > 1 ? 256 : 1];
    const int head = blockIdx.x % a.p.kv_heads;
    Item it;
    if (!find<ROWS, KEYS, true>(a, blockIdx.x / a.p.kv_heads, target, it)) return;
    if ((it.slot + it.splits - 1) * a.p.kv_heads + head >= a.slots) return;
    const float *ml = a.partial + a.slots * ROWS * D;
    const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave, group = threadIdx.x / kItems % kGroups;
    const int rows = min(it.run.n * a.group - it.tile * ROWS, ROWS);
    for (int first = blockIdx.y * MINE; first < rows; first += gridDim.y * MINE) {
        const int row0 = it.tile * ROWS + first, used = min(rows - first, MINE);
        auto place = [&](int s, int r) { return ((it.slot + s) * a.p.kv_heads + head) * ROWS + first + r; };
        f32x4 o[(kItems + 255) / 256];
#pragma unroll
        for (int k = 0; k < (kItems + 255) / 256; ++k) o[k] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        __syncthreads();                         // (what the rows in front of these have left)
        // maxima and sums of rows: a wave a row
        for (int r = wave; r < used; r += 4) {
            float m = -INFINITY, l = 0.0f;
            for (int s = lane; s < it.splits; s += kWave) m = fmaxf(m, ml[place(s, r) * 2]);
#pragma unroll
            for (int off = kWave / 2; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor(m, off, kWave));
            for (int s = lane; s < it.splits; s += kWave) l = __fmaf_rn(ml[place(s, r) * 2 + 1], weight_of(ml[place(s, r) * 2], m), l);
            l = wave_add(l);
            if (lane == 0) tops[r] = m, totals[r] = l;
        }
        for (int s0 = 0; s0 < it.splits; s0 += kSplits) {
            const int count = min(kSplits, it.splits - s0);
            __syncthreads();
            for (int e = threadIdx.x; e < used * count; e += 256) weight[e / count][e % count] = weight_of(ml[place(s0 + e % count, e / count) * 2], tops[e / count]);
            __syncthreads();
#pragma unroll
            for (int k = 0; k < (kItems + 255) / 256; ++k) {
                const int e = kGroups > 1 ? threadIdx.x % kItems : threadIdx.x + k * 256, r = e / kColumns, d = e % kColumns * 4;
                if (r >= used) continue;
                const float *from = a.partial + place(s0, r) * D + d;
                const int64_t step = (int64_t)a.p.kv_heads * ROWS * D;
#pragma unroll 4
                for (int s = group; s < count; s += kGroups) o[k] += *reinterpret_cast<const f32x4 *>(from + s * step) * weight[r][s];
            }
        }
        if constexpr (kGroups > 1) {
            part[threadIdx.x] = o[0];
            __syncthreads();
#pragma unroll
            for (int g = 1; g < kGroups; ++g)
                if (!group) o[0] += part[threadIdx.x + g * kItems];
        }
#pragma unroll
        for (int k = 0; k < (kItems + 255) / 256; ++k) {
            const int e = threadIdx.x + k * 256, r = e / kColumns, d = e % kColumns * 4;
            if (r < used && d < a.p.dim && (kGroups == 1 || !group)) store_row(a, it.run, row0 + r, head, d, answer_of(o[k], totals[r], quotient_of(a, head, totals[r])));
        }
    }
}

// ---------------------------------------------------------------------------------------------------------------- host
// What a call launches: which sequences go to which kernel, and what they need.
struct Plan {
    bool few, many;
    int least;                                   // rows a key head from which on (exclusive) the kernel for many has them
};
Plan plan_of(int64_t group, int64_t rows, int64_t seqs, int64_t most_new) {
    if (most_new * group <= kFewRows) return {true, false, 0};
    if (seqs <= 1 || rows >= seqs * most_new) return {false, true, 0};        // (all of them alike: none has few)
    return {true, true, kFewRows};
}
int64_t slots_of(int target) { return 2 * target; }
int64_t floats_of(int rows, int target, int D) { return slots_of(target) * rows * (D + 2); }

}  // namespace
}  // namespace odl

using namespace odl;

namespace {

int check(const char *who, int64_t heads, int64_t most_new, const odl_fp8_paged_cache *cache, const odl_fp8_paged_batch *batch, Paged &p) {
    if (const int rc = take_paged(who, cache, batch, p)) return rc;
    if (heads < 1 || heads > 1024 || heads % p.kv_heads) return set_error(ODL_ERR_SHAPE, "%s: %lld heads for %d of keys (a multiple, up to 1024)", who, (long long)heads, p.kv_heads);
    if (batch->rows * heads >= INT32_MAX) return set_error(ODL_ERR_SHAPE, "%s: more than 2^31 rows of heads", who);
    if (most_new < 0) return set_error(ODL_ERR_ARG, "%s: most_new is negative", who);
    return ODL_OK;
}

template <int D, int C, bool CAP>
int launch(Attend &a, const Plan &plan, int64_t most_rows, float *workspace, hipStream_t stream) {
    const int64_t kv = a.p.kv_heads, rows = (int64_t)a.p.rows * a.group, seqs = a.p.seqs < a.p.rows ? a.p.seqs : a.p.rows;
    // no more tiles than sequences (those that fill no tile) and rows / tile; splits that begin anew: see `find`
    auto blocks = [&](int64_t tiles, int target) { return (target / kv + 1 + tiles) * kv; };
    auto joins = [&](int target) { return (unsigned)((target / kv + 1) * kv); };
    const int few = few_target(D, a.p.e4m3);
    const int64_t many_blocks = blocks(seqs + rows / kManyRows, kManyTarget), few_blocks = blocks(plan.many ? seqs : seqs + rows / kFewRows, few);         // (beside the other kernel: a tile a sequence)
    if ((plan.many && many_blocks * kManyWaves * kWave > UINT32_MAX) || (plan.few && few_blocks * kFewWaves * kWave > UINT32_MAX))
        return set_error(ODL_ERR_SHAPE, "odl_fp8_paged_attention: more tiles of rows than a launch has blocks (times key heads, below 2^24 of few rows and 2^23 of many)");
    if (plan.many) {
        a.least_rows = plan.least, a.most_rows = INT32_MAX;
        a.partial = workspace, a.slots = slots_of(kManyTarget);
        const int clear = !plan.few;
        const dim3 grid((unsigned)many_blocks);
        if (a.p.e4m3) hipLaunchKernelGGL((attend_many_kernel<D, C, true, CAP>), grid, dim3(kManyWaves * kWave), many_lds(D), stream, a, clear);
        else hipLaunchKernelGGL((attend_many_kernel<D, C, false, CAP>), grid, dim3(kManyWaves * kWave), many_lds(D), stream, a, clear);
        if (a.p.reach > kManyKeys)
            hipLaunchKernelGGL((attend_join_kernel<D, kManyRows, kManyKeys, kJoinMany>), dim3(joins(kManyTarget), kManyRows / kJoinMany), dim3(256), 0, stream, a, (uint32_t)kManyTarget);
        workspace += floats_of(kManyRows, kManyTarget, D);
    }
    if (plan.few) {
        a.least_rows = 0, a.most_rows = plan.many ? plan.least : INT32_MAX;
        a.partial = workspace, a.slots = slots_of(few);
        const dim3 grid((unsigned)few_blocks);
        if (a.p.e4m3) hipLaunchKernelGGL((attend_few_kernel<D, true, CAP>), grid, dim3(kFewWaves * kWave), few_lds(D, true), stream, a);
        else hipLaunchKernelGGL((attend_few_kernel<D, false, CAP>), grid, dim3(kFewWaves * kWave), few_lds(D, false), stream, a);
        if (a.p.reach > kUncut * kFewKeys * kFewWaves)
            hipLaunchKernelGGL((attend_join_kernel<D, kFewRows, kFewKeys * kFewWaves, kJoinFew>), dim3(joins(few), (unsigned)(((most_rows < kFewRows ? most_rows : kFewRows) + kJoinFew - 1) / kJoinFew)), dim3(256), 0, stream, a,
                               (uint32_t)few);
    }
    return check_launch("odl_fp8_paged_attention");
}

int64_t workspace_of(const Plan &plan, const Paged &p) {
    const int D = p.dim > 64 ? 128 : 64;
    return (plan.many ? floats_of(kManyRows, kManyTarget, D) : 0) + (plan.few ? floats_of(kFewRows, few_target(D, p.e4m3), D) : 0);
}

}  // namespace

extern "C" int64_t odl_fp8_paged_attention_workspace(int64_t heads, int64_t most_new, const odl_fp8_paged_cache *cache, const odl_fp8_paged_batch *batch) {
    Paged p;
    if (check("odl_fp8_paged_attention_workspace", heads, most_new, cache, batch, p)) return -1;
    return workspace_of(plan_of(heads / p.kv_heads, p.rows, p.seqs, most_new < p.rows ? most_new : p.rows), p);
}

extern "C" int odl_fp8_paged_attention(const void *q, const int64_t *q_strides, int64_t heads, int64_t most_new, const odl_fp8_paged_cache *cache,
                                       const odl_fp8_paged_batch *batch, float scale, int64_t window, float softcap, void *out, float *workspace,
                                       int64_t workspace_floats, odl_stream_t stream_) {
    static const char who[] = "odl_fp8_paged_attention";
    Attend a;
    if (const int rc = check(who, heads, most_new, cache, batch, a.p)) return rc;
    if (const int rc = check_strides(who, "q", q, q_strides, a.p.rows)) return rc;
    if (!(scale > 0.0f) || scale > 1e30f) return set_error(ODL_ERR_ARG, "%s: scale %g (above 0, up to 1e30)", who, (double)scale);
    if (!(softcap == 0.0f || (softcap >= 1e-3f && softcap <= 1e6f))) return set_error(ODL_ERR_ARG, "%s: softcap %g (0, or 1e-3 to 1e6)", who, (double)softcap);
    if (window < 0) return set_error(ODL_ERR_ARG, "%s: window %lld", who, (long long)window);
    if (a.p.rows == 0) return ODL_OK;
    if (!out || (reinterpret_cast<uintptr_t>(out) & 15)) return set_error(ODL_ERR_ARG, "%s: out must be a 16-byte aligned address", who);
    a.q = static_cast<const uint16_t *>(q), a.q_row = q_strides[0], a.q_head = q_strides[1];
    a.heads = (int)heads, a.group = (int)(heads / a.p.kv_heads), a.window = window == 0 || window > INT32_MAX / 2 ? INT32_MAX / 2 : (int)window;
    a.scale = scale, a.softcap = softcap, a.out = static_cast<uint16_t *>(out);
    const Plan plan = plan_of(a.group, a.p.rows, a.p.seqs, most_new < a.p.rows ? most_new : a.p.rows);
    if (!workspace || workspace_floats < workspace_of(plan, a.p) || (reinterpret_cast<uintptr_t>(workspace) & 15))
        return set_error(ODL_ERR_ARG, "%s: a workspace of %lld floats, 16-byte aligned", who, (long long)workspace_of(plan, a.p));
    hipStream_t stream = reinterpret_cast<hipStream_t>(stream_);
    const int64_t most_rows = (most_new < 1 ? 1 : most_new < a.p.rows ? most_new : a.p.rows) * a.group;
    // heads of up to 96: a quarter of the products of 128 less (the prompts above 206 -> 192 us; the kernel for few rows waits for memory, and has one form)
    // Kernels with a cap are apart: its code in the loop costs the others 1 to 4 per cent (one token behind 200, 12 heads of 64: 7.9 and 8.2 us; the chunk above 519 and 527).
#define ODL_ATTEND(D, C) (softcap > 0.0f ? launch<D, C, true>(a, plan, most_rows, workspace, stream) : launch<D, C, false>(a, plan, most_rows, workspace, stream))
    return a.p.dim > 96 ? ODL_ATTEND(128, 128) : a.p.dim > 64 ? ODL_ATTEND(128, 96) : ODL_ATTEND(64, 64);
#undef ODL_ATTEND
}
