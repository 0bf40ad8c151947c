// Log probabilities of given tokens from the logits of a head, with the entropy of each row and its top alternatives, and the
// gradient of the logits.  With d_j = (l_j - m) / T, m the row's maximum, s = sum e^d_j, q = sum e^d_j d_j:
//   logprob = d_t - ln s,  entropy = ln s - q / s (both terms >= 0: nothing cancels),  top_i = d_i - ln s
//   p_j = e^d_j / s,  dl_j = [A (j == t) + sum_i C_i (j == id_i) - p_j (A + sum_i C_i) - B p_j (ln p_j + entropy)] / T
// for gradients A of the logprob, B of the entropy, C_i of the top alternatives.
//
// The forward reads a row once, a block a row or a part of it, with a running maximum and the two sums of it per lane.  The top k cost no work in that
// pass: the lanes' maxima are folded to 64 (or, for many alternatives, searched bit by bit), the k-th largest of those is a lower bound of the k-th
// largest logit, and only lanes whose maximum reaches it can hold one; their share of the row is read again and what reaches the bound is ranked.
// Rows are read and written with 16-byte accesses at any alignment (rows of an odd number of columns begin anywhere).
// Bound by HBM for large calls (8 to 12 operations an element, one of them an exponential), by latency for a few rows.  8192 x 50257 bf16: forward
// 155 to 165 us (5.0 to 5.3 TB/s), backward 340 us (4.8 TB/s read and written); 2048 rows with the top 5 47 us (4.3); 1004 rows of fp32 at odd addresses
// 50 (4.1) and 74; 16 rows of 32000 with the top 20 9.5.  A row is one block's, but for few
// rows of a large vocabulary, which are cut over several blocks and joined by a second launch (parts_of).
#include "common.h"

#pragma clang fp contract(off)

namespace odl {
namespace {

constexpr int kParts = ODL_FP8_AMAX_PARTS;
constexpr int kMaxTop = ODL_FP8_LOGPROBS_MAX_TOP;
constexpr int kCand = 1024;                      // candidates that are ranked at once
constexpr int kMaxParts = 16;                    // (their top k are ranked at once)
constexpr int kFolded = 32;                      // up to so many alternatives 64 folded maxima give a good bound
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kFar = 1e30f;                    // exponents are cut off here: finite times e^-far is 0, infinity times 0 is not
constexpr float kGone = 256.0f;                  // and here in the backward: 2^-256 is 0 as well, and times a factor of up to 2^119 the exponent stays finite

template <int DT> struct Elem;
template <> struct Elem<ODL_BF16> { typedef uint16_t T; static constexpr int vecs = 1; };
template <> struct Elem<ODL_F32> { typedef float T; static constexpr int vecs = 2; };

template <int DT>
__device__ __forceinline__ float one(const typename Elem<DT>::T *p) {
    if constexpr (DT == ODL_BF16) return bits_to_float((uint32_t)*p << 16);
    else return *p;
}

// eight elements from any address that suits one of them
template <int DT>
struct Chunk {
    u32x4 raw[Elem<DT>::vecs];
    __device__ __forceinline__ void load(const typename Elem<DT>::T *p) { __builtin_memcpy(raw, p, sizeof(raw)); }
    __device__ __forceinline__ void fill() {     // -inf: weighs nothing
#pragma unroll
        for (int v = 0; v < Elem<DT>::vecs; ++v) raw[v] = DT == ODL_BF16 ? u32x4{0xff80ff80u, 0xff80ff80u, 0xff80ff80u, 0xff80ff80u}
                                                                         : u32x4{0xff800000u, 0xff800000u, 0xff800000u, 0xff800000u};
    }
    __device__ __forceinline__ void widen(float (&f)[8]) const {
        if constexpr (DT == ODL_BF16) {
#pragma unroll
            for (int q = 0; q < 4; ++q) { f[2 * q] = bf16_lo(raw[0][q]); f[2 * q + 1] = bf16_hi(raw[0][q]); }
        } else {
#pragma unroll
            for (int q = 0; q < 8; ++q) f[q] = bits_to_float(raw[q / 4][q % 4]);
        }
    }
};

// The exponent of an element, in powers of two, against a running maximum m: d = (l - m) * c, c = log2(e) / T.  With mc = m * c rounded it is one
// fused multiply-add, l * c - mc: the rounding of mc is the same for every element and for the maximum itself, so nothing is lost by
// it as long as sums are held against mc and not against m.  It moves every exponent by up to 2^-25 |mc|, though, and the sums by as many
// powers of two: maxima beyond 2^24, where that is more than a half, take the difference first, and sums are held against m * c itself.
struct Exponent {
    float m, mc, c;
    bool near;
    __device__ __forceinline__ Exponent(float m_, float c_) : m(m_), mc(m_ * c_), c(c_), near(__builtin_fabsf(m_ * c_) < 0x1p24f) {}
    __device__ __forceinline__ float operator()(float l) const { return near ? __fmaf_rn(l, c, -mc) : (l - m) * c; }
};

// How far down it is from what is held against maximum m to what is held against `to` (and finite: what was summed against m is 0 then).
__device__ __forceinline__ float descent(float m, float to, float c) {
    const Exponent a(m, c), b(to, c);
    const float down = a.near ? (b.near ? b.mc - a.mc : __fmaf_rn(to, c, -a.mc)) : (b.near ? -__fmaf_rn(m, c, -b.mc) : (to - m) * c);
    return fminf(down, kFar);
}

// sums over a wave, in every lane
template <int CTRL>
__device__ __forceinline__ float add_dpp(float v) {
    return v + bits_to_float((uint32_t)__builtin_amdgcn_update_dpp(0, (int)float_to_bits(v), CTRL, 0xf, 0xf, false));
}
__device__ __forceinline__ float wave_sum(float v) {
    v = add_dpp<0xB1>(v);                        // lane ^ 1, ^ 2, the other quad of 8, the other half of 16
    v = add_dpp<0x4E>(v);
    v = add_dpp<0x141>(v);
    v = add_dpp<0x140>(v);
    const auto r = __builtin_amdgcn_permlane16_swap(float_to_bits(v), float_to_bits(v), false, false);
    v = bits_to_float(r[0]) + bits_to_float(r[1]);
    const auto q = __builtin_amdgcn_permlane32_swap(float_to_bits(v), float_to_bits(v), false, false);
    return bits_to_float(q[0]) + bits_to_float(q[1]);
}
template <int CTRL>
__device__ __forceinline__ float max_dpp(float v) {
    return fmaxf(v, bits_to_float((uint32_t)__builtin_amdgcn_update_dpp(0, (int)float_to_bits(v), CTRL, 0xf, 0xf, false)));
}
// maxima over groups of 4, 8 or 64 lanes
template <int LANES>
__device__ __forceinline__ float group_max(float v) {
    v = max_dpp<0x4E>(max_dpp<0xB1>(v));
    if constexpr (LANES >= 8) v = max_dpp<0x141>(v);
    if constexpr (LANES >= 64) {
        v = max_dpp<0x140>(v);
        const auto r = __builtin_amdgcn_permlane16_swap(float_to_bits(v), float_to_bits(v), false, false);
        v = fmaxf(bits_to_float(r[0]), bits_to_float(r[1]));
        const auto q = __builtin_amdgcn_permlane32_swap(float_to_bits(v), float_to_bits(v), false, false);
        v = fmaxf(bits_to_float(q[0]), bits_to_float(q[1]));
    }
    return v;
}

struct Row {                                     // what a row answers: its maximum, log2 of the sum against it, its entropy
    float m, log2_s, entropy;
};

__device__ __forceinline__ float log_prob(float l, const Row &r, float c) {
    if (r.log2_s == -INFINITY) return -INFINITY; // every logit is -inf
    return (Exponent(r.m, c)(l) - r.log2_s) * kLn2;
}

// A float as a number that is larger where it is (no NaN), and the least float whose number has these upper 16 bits.
__device__ __forceinline__ uint32_t order_key(float v) {
    const uint32_t u = float_to_bits(v);
    return u >> 31 ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float order_least(uint32_t upper) {
    const uint32_t key = upper << 16;
    return fmaxf(bits_to_float(key >> 31 ? key & 0x7fffffffu : ~key), -INFINITY);          // (below -inf: all of them)
}

__device__ __forceinline__ bool before(float v, int i, float w, int j) { return v > w || (v == w && i < j); }

struct Forward {
    const void *logits;
    const int64_t *targets;
    int64_t rows, stride, ignore_index;
    int vocab, top_k;
    float c;                                     // log2(e) / T
    float *logprobs, *entropy, *stats, *top_logprobs;
    int64_t *top_ids;
    float *partial;                              // of rows that several blocks share: [rows][parts][3 + 2 top_k]
    int parts, span;                             // parts of a row, columns of one (a multiple of 8)
};

// A row that is not read.
__device__ __forceinline__ void ignored(const Forward &a, int64_t row, int tid) {
    if (tid == 0) {
        a.logprobs[row] = 0.0f;
        a.entropy[row] = 0.0f;
        if (a.stats) { a.stats[row] = 0.0f; a.stats[a.rows + row] = 0.0f; }
    }
    if (tid < a.top_k) {
        a.top_logprobs[row * a.top_k + tid] = 0.0f;
        a.top_ids[row * a.top_k + tid] = -1;
    }
}

// What sum and weighted sum against the maximum say.
__device__ __forceinline__ Row row_of(float m, float s, float q) {
    Row r;
    r.m = m;
    r.log2_s = s == 0.0f ? -INFINITY : log2f(s);
    r.entropy = s == 0.0f ? 0.0f : (r.log2_s - q / s) * kLn2;
    return r;
}

template <int DT>
__device__ __forceinline__ void answer(const Forward &a, int64_t row, int64_t target, const Row &r) {
    const typename Elem<DT>::T *p = reinterpret_cast<const typename Elem<DT>::T *>(a.logits) + row * a.stride;
    a.logprobs[row] = target >= 0 && target < a.vocab ? log_prob(one<DT>(p + target), r, a.c) : __builtin_nanf("");
    a.entropy[row] = r.entropy;
    if (a.stats) { a.stats[row] = r.m; a.stats[a.rows + row] = r.log2_s; }
}

// An alternative of its rank; a row with NaN or +inf has no order.
__device__ __forceinline__ void alternative(const Forward &a, int64_t row, const Row &r, int rank, float v, int id) {
    const bool sound = r.log2_s == r.log2_s;
    a.top_logprobs[row * a.top_k + rank] = sound ? log_prob(v, r, a.c) : __builtin_nanf("");
    a.top_ids[row * a.top_k + rank] = sound ? id : -1;
}

// How many of n candidates come before (v, id).  The arrays are filled up to a multiple of 8 with what comes before nothing.
__device__ __forceinline__ int rank_of(const float *values, const int *ids, int n, float v, int id) {
    int rank = 0;
    for (int j = 0; j < n; j += 8) {
        float w[8];
        int i[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) { w[u] = values[j + u]; i[u] = ids[j + u]; }
#pragma unroll
        for (int u = 0; u < 8; ++u) rank += before(w[u], i[u], v, id);
    }
    return rank;
}

// PART: a block has one of the parts of a row, and leaves its maximum, its sums and its top k for the join.
template <int DT, int THREADS, bool PART>
__global__ __launch_bounds__(THREADS) void token_logprobs_kernel(const Forward a) {
    typedef typename Elem<DT>::T T;
    constexpr int U = 4, kWaves = THREADS / kWave;
    __shared__ float wave_m[kWaves], wave_s[kWaves], wave_q[kWaves], cand_v[kCand];
    __shared__ __attribute__((aligned(16))) float group_top[THREADS];
    __shared__ int cand_i[kCand], lanes[THREADS], n_lanes, n_cand;
    const int tid = threadIdx.x, lane = tid % kWave;
    const int64_t row = blockIdx.x;
    const int64_t target = a.targets[row];
    if (target == a.ignore_index) {
        if (!PART) ignored(a, row, tid);
        return;
    }
    const int first = PART ? (int)blockIdx.y * a.span : 0, end = PART ? min(first + a.span, a.vocab) : a.vocab;
    float *mine = a.partial + (row * a.parts + blockIdx.y) * (3 + 2 * a.top_k);
    const T *p = reinterpret_cast<const T *>(a.logits) + row * a.stride + first;
    const int n = (end - first) / 8, tail = (end - first) % 8;
    // running maximum (never below -FLT_MAX, so that differences from it are finite or -inf), sum 2^d, sum 2^d d
    float m = -FLT_MAX, s = 0.0f, q = 0.0f, top = -INFINITY;
    auto move_to = [&](float to) {
        const float down = descent(m, to, a.c), f = __builtin_amdgcn_exp2f(-down);
        q = f * __fmaf_rn(-down, s, q);
        s *= f;
        m = to;
    };
    for (int i = tid; i < n; i += U * THREADS) {
        Chunk<DT> in[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (i + u * THREADS < n) in[u].load(p + (int64_t)(i + u * THREADS) * 8);
            else in[u].fill();
        }
        float f[U][8], most = -INFINITY;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            in[u].widen(f[u]);
#pragma unroll
            for (int e = 0; e < 8; ++e) most = fmaxf(most, f[u][e]);
        }
        if (most > top) {                        // (rare behind the first trips; -inf and NaN move nothing)
            top = most;
            move_to(fmaxf(m, most));
        }
        const Exponent x(m, a.c);
        if (x.near) {
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float d = __fmaf_rn(f[u][e], x.c, -x.mc), w = __builtin_amdgcn_exp2f(d);
                    s += w;
                    q = __fmaf_rn(w, fmaxf(d, -kFar), q);
                }
        } else {
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float d = (f[u][e] - m) * x.c, w = __builtin_amdgcn_exp2f(d);
                    s += w;
                    q = __fmaf_rn(w, fmaxf(d, -kFar), q);
                }
        }
    }
    if (tid < tail) {
        const float l = one<DT>(p + n * 8 + tid);
        top = fmaxf(top, l);
        move_to(fmaxf(m, l));
        const float d = Exponent(m, a.c)(l), w = __builtin_amdgcn_exp2f(d);
        s += w;
        q = __fmaf_rn(w, fmaxf(d, -kFar), q);
    }
    // the block's maximum, every lane's sums against it, their sums
    const float wm = group_max<kWave>(m);
    if (lane == 0) wave_m[tid / kWave] = wm;
    if (a.top_k) {
        if (a.top_k <= kFolded) {
            const float g = group_max<THREADS / kWave>(top);
            if (tid % (THREADS / kWave) == 0) group_top[tid / (THREADS / kWave)] = g;
        } else {
            group_top[tid] = top;
        }
        if (tid == 0) n_lanes = n_cand = 0;
    }
    __syncthreads();
    float to = wave_m[0];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) to = fmaxf(to, wave_m[w]);
    move_to(to);
    const float ws = wave_sum(s), wq = wave_sum(q);
    if (lane == 0) { wave_s[tid / kWave] = ws; wave_q[tid / kWave] = wq; }
    float least = 0.0f;
    if (a.top_k > kFolded) {
        // a bound of the k-th largest of all lanes' maxima: the largest number of 16 bits that k of them reach, bit by bit
        uint32_t key[THREADS / kWave], reach = 0;
#pragma unroll
        for (int j = 0; j < THREADS / kWave; ++j) key[j] = order_key(group_top[j * kWave + lane]) >> 16;
        for (uint32_t bit = 1u << 15; bit; bit >>= 1) {
            int count = 0;
#pragma unroll
            for (int j = 0; j < THREADS / kWave; ++j) count += __popcll(__ballot(key[j] >= (reach | bit)));
            if (count >= a.top_k) reach |= bit;
        }
        least = order_least(reach);
        if (top >= least) lanes[atomicAdd(&n_lanes, 1)] = tid;
    } else if (a.top_k) {                        // the k-th largest of the 64 maxima; every wave finds it for itself
        const float v = group_top[lane];
        int above = 0, equal = 0;
#pragma unroll
        for (int j = 0; j < kWave; j += 4) {
            const float4 o = *reinterpret_cast<const float4 *>(group_top + j);
            above += (o.x > v) + (o.y > v) + (o.z > v) + (o.w > v);
            equal += (o.x == v) + (o.y == v) + (o.z == v) + (o.w == v);
        }
        const uint64_t kth = __ballot(above < a.top_k && a.top_k <= above + equal);
        least = __shfl(v, __ffsll((unsigned long long)kth) - 1, kWave);
        if (top >= least) lanes[atomicAdd(&n_lanes, 1)] = tid;
    }
    __syncthreads();
    s = wave_s[0];
    q = wave_q[0];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) { s += wave_s[w]; q += wave_q[w]; }
    const Row r = row_of(m, s, q);
    if (tid == 0) {
        if constexpr (PART) { mine[0] = m; mine[1] = s; mine[2] = q; }
        else answer<DT>(a, row, target, r);
    }
    if (!a.top_k) return;

    auto put = [&](int rank, float v, int id) {
        if constexpr (PART) { mine[3 + rank] = v; reinterpret_cast<uint32_t *>(mine)[3 + a.top_k + rank] = (uint32_t)first + (uint32_t)id; }
        else alternative(a, row, r, rank, v, id);
    };
    auto offer = [&](float v, int col) {
        if (v >= least) {
            const int at = atomicAdd(&n_cand, 1);
            if (at < kCand) { cand_v[at] = v; cand_i[at] = col; }
        }
    };
    const int per = (n + THREADS - 1) / THREADS, total = n_lanes * per;
    for (int i = tid; i < total; i += THREADS) {
        const int chunk = lanes[i / per] + (i % per) * THREADS;
        if (chunk < n) {
            Chunk<DT> in;
            in.load(p + (int64_t)chunk * 8);
            float f[8];
            in.widen(f);
#pragma unroll
            for (int e = 0; e < 8; ++e) offer(f[e], chunk * 8 + e);
        }
    }
    if (tid < tail) offer(one<DT>(p + n * 8 + tid), n * 8 + tid);
    __syncthreads();
    const int found = n_cand;
    if (found <= kCand) {
        if (tid < 8 && found + tid < kCand) { cand_v[found + tid] = -INFINITY; cand_i[found + tid] = INT_MAX; }
        __syncthreads();
        for (int i = tid; i < found; i += THREADS) {
            const float v = cand_v[i];
            const int id = cand_i[i], rank = rank_of(cand_v, cand_i, found, v, id);
            if (rank < a.top_k) put(rank, v, id);
        }
        if (tid >= found && tid < a.top_k) put(tid, -INFINITY, 0);         // (fewer than k: NaN in the row, which has no order)
        return;
    }
    // More than a thousand logits share the bound (rows with fewer allowed logits than alternatives are asked for, say): the largest behind the
    // last one found, k times over, a read of the row each: 16 x 32000 with 10 logits that are not masked, top 20, 116 us, top 64 335 (no mask: 9 and 12).
    float last_v = INFINITY;
    int last_i = -1;
    for (int k = 0; k < a.top_k; ++k) {
        float best_v = -INFINITY;
        int best_i = INT_MAX;
        auto look = [&](float v, int id) {
            if (before(last_v, last_i, v, id) && before(v, id, best_v, best_i)) { best_v = v; best_i = id; }
        };
        for (int i = tid; i < n; i += THREADS) {
            Chunk<DT> in;
            in.load(p + (int64_t)i * 8);
            float f[8];
            in.widen(f);
#pragma unroll
            for (int e = 0; e < 8; ++e) look(f[e], i * 8 + e);
        }
        if (tid < tail) look(one<DT>(p + n * 8 + tid), n * 8 + tid);
#pragma unroll
        for (int off = kWave / 2; off > 0; off >>= 1) {
            const float v = __shfl_xor(best_v, off, kWave);
            const int id = __shfl_xor(best_i, off, kWave);
            if (before(v, id, best_v, best_i)) { best_v = v; best_i = id; }
        }
        __syncthreads();                         // (cand_v and cand_i are read by everybody in the round before)
        if (lane == 0) { cand_v[tid / kWave] = best_v; cand_i[tid / kWave] = best_i; }
        __syncthreads();
        best_v = cand_v[0];
        best_i = cand_i[0];
        for (int w = 1; w < kWaves; ++w)
            if (before(cand_v[w], cand_i[w], best_v, best_i)) { best_v = cand_v[w]; best_i = cand_i[w]; }
        last_v = best_v;
        last_i = best_i;
        if (tid == 0) put(k, best_v, best_i);
    }
}

// Rows that several blocks share: the maxima and sums of their parts and the largest of their top k.  Each part has at least
// ceil(k / parts) logits that reach its own one of that rank, and k that reach its last: the smallest of the former and the largest of the latter are bounds
// of the k-th largest of the row, and little more than k candidates reach them.
template <int DT>
__global__ __launch_bounds__(256) void token_logprobs_join_kernel(const Forward a) {
    __shared__ float cand_v[kCand];
    __shared__ int cand_i[kCand], n_cand;
    const int tid = threadIdx.x, record = 3 + 2 * a.top_k;
    const int64_t row = blockIdx.x, target = a.targets[row];
    if (target == a.ignore_index) return ignored(a, row, tid);
    const float *from = a.partial + row * a.parts * record;
    if (tid == 0) n_cand = 0;
    // a part a lane, sixteen lanes at a time; every wave for itself
    const bool have = tid % 16 < a.parts;
    const float *part = from + tid % 16 * record;
    const float pm = have ? part[0] : -FLT_MAX, ps = have ? part[1] : 0.0f, pq = have ? part[2] : 0.0f;
    float m = pm, each = INFINITY, last = -INFINITY;
    if (have && a.top_k) {
        each = part[3 + (a.top_k + a.parts - 1) / a.parts - 1];
        last = part[3 + a.top_k - 1];
    }
    static_assert(kMaxParts == 16, "a group of lanes has the parts");
#pragma unroll
    for (int off = 8; off > 0; off >>= 1) {
        m = fmaxf(m, __shfl_xor(m, off, kWave));
        each = fminf(each, __shfl_xor(each, off, kWave));
        last = fmaxf(last, __shfl_xor(last, off, kWave));
    }
    const float least = fmaxf(each, last), down = descent(pm, m, a.c), f = __builtin_amdgcn_exp2f(-down);
    float s = f * ps, q = f * __fmaf_rn(-down, ps, pq);
#pragma unroll
    for (int off = 8; off > 0; off >>= 1) {
        s += __shfl_xor(s, off, kWave);
        q += __shfl_xor(q, off, kWave);
    }
    __syncthreads();
    for (int i = tid; i < a.parts * a.top_k; i += 256) {
        const float *at = from + i / a.top_k * record + 3 + i % a.top_k;
        const float v = at[0];
        const int id = reinterpret_cast<const int *>(at)[a.top_k];
        if (v >= least) {
            const int to = atomicAdd(&n_cand, 1);
            cand_v[to] = v;
            cand_i[to] = id;
        }
    }
    const Row r = row_of(m, s, q);
    if (tid == 0) answer<DT>(a, row, target, r);
    __syncthreads();
    const int n = n_cand;
    if (r.log2_s != r.log2_s) {                  // (candidates of such a row may be fewer)
        if (tid < a.top_k) alternative(a, row, r, tid, 0.0f, 0);
        return;
    }
    if (tid < 8 && n + tid < kCand) { cand_v[n + tid] = -INFINITY; cand_i[n + tid] = INT_MAX; }
    __syncthreads();
    for (int i = tid; i < n; i += 256) {
        const int rank = rank_of(cand_v, cand_i, n, cand_v[i], cand_i[i]);
        if (rank < a.top_k) alternative(a, row, r, rank, cand_v[i], cand_i[i]);
    }
}

struct Backward {
    const void *logits;
    const int64_t *targets, *top_ids;
    const float *d_logprobs, *d_entropy, *d_top, *stats, *entropy;
    int64_t rows, stride, ignore_index, items;
    int vocab, padded, top_k, sections, section;  // sections of a row, columns of one (a multiple of 8)
    float inv_t;
    void *dlogits;
    float *parts;
};

// 1024 lanes keep more of a row on its way than 512: 8192 x 50304 bf16 388 -> 347 us (2 sections a row; with stores that bypass the caches 338, but then
// the cast behind finds nothing there, and 1004 x 50257 fp32 goes 86 -> 89)
constexpr int kBwdThreads = 1024, kMarks = 128;

// An item is a section of a row; blocks take them round-robin (at most one block for each partial maximum).
template <int DT, bool TOP>
__global__ __launch_bounds__(kBwdThreads) void token_logprobs_bwd_kernel(const Backward a) {
    typedef typename Elem<DT>::T T;
    constexpr int U = 4;
    __shared__ uint32_t red[kBwdThreads / kWave], marks[TOP ? kMarks : 1];
    __shared__ float top_d[TOP ? kMaxTop : 1];
    __shared__ int top_i[TOP ? kMaxTop : 1];
    const int tid = threadIdx.x;
    uint32_t am = 0;                             // bf16: a packed pair of magnitudes
    for (int64_t item = blockIdx.x; item < a.items; item += gridDim.x) {
        const int64_t row = item / a.sections;
        const int first = (int)(item - row * a.sections) * a.section, end = min(first + a.section, a.padded);
        const T *in = reinterpret_cast<const T *>(a.logits) + row * a.stride;
        T *out = reinterpret_cast<T *>(a.dlogits) + row * a.padded;
        const int64_t target = a.targets[row];
        const float l2 = a.stats[a.rows + row];
        const Exponent x(a.stats[row], a.inv_t * kLog2e);
        const bool nothing = target == a.ignore_index || l2 == -INFINITY;
        const float of_logprob = a.d_logprobs ? a.d_logprobs[row] : 0.0f, b = a.d_entropy ? a.d_entropy[row] : 0.0f, entropy = a.entropy[row];
        float sum = of_logprob, reach = __builtin_fabsf(of_logprob) + __builtin_fabsf(b) * (kGone + entropy);
        if constexpr (TOP) {
            __syncthreads();                     // the item before has been read
            for (int i = tid; i < kMarks; i += kBwdThreads) marks[i] = 0;
            __syncthreads();
            if (tid < a.top_k) {
                const int id = (int)a.top_ids[row * a.top_k + tid];
                top_i[tid] = id;
                top_d[tid] = a.d_top[row * a.top_k + tid];
                if (id >= 0) atomicOr(&marks[(id / 8 / 32) % kMarks], 1u << (id / 8 % 32));
            }
            __syncthreads();
            for (int i = 0; i < a.top_k; ++i) {
                sum += top_d[i];
                reach += __builtin_fabsf(top_d[i]);
            }
        }
        // gradient of an element = p * (k0 + k1 * log2 p).  Factors that 1 / T would take out of range (0 times infinity is not 0) are left without
        // it, and it is multiplied onto the products.
        const bool late = !(reach * a.inv_t < 1e38f);
        const float by = late ? 1.0f : a.inv_t, given = of_logprob * by;
        float k0 = -by * __fmaf_rn(b, entropy, sum);
        const float k1 = -by * b * kLn2;
        if (target < 0 || target >= a.vocab) k0 = __builtin_nanf("");          // no such token: its log probability is NaN too
        const int t_chunk = target >= 0 && target < a.vocab ? (int)target / 8 : -1;
        auto gradient = [&](float l) {
            const float y = x(l) - l2;
            return __builtin_amdgcn_exp2f(y) * __fmaf_rn(fmaxf(y, -kGone), k1, k0);
        };
        // gradients of a chunk in which the target or a top alternative may lie, or that ends behind the vocabulary
        auto special = [&](int chunk, float (&f)[8]) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int col = chunk * 8 + e;
                if (chunk == t_chunk && col == (int)target) f[e] += given;
                if constexpr (TOP)
                    for (int i = 0; i < a.top_k; ++i)
                        if (top_i[i] == col) f[e] = __fmaf_rn(top_d[i], by, f[e]);
                if (col >= a.vocab) f[e] = 0.0f;
            }
        };
        auto store = [&](int chunk, const float (&f)[8]) {
            if constexpr (DT == ODL_BF16) {
                const u32x4 w = {pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7])};
#pragma unroll
                for (int q = 0; q < 4; ++q) am = max_u16x2(am, abs_bf16x2(w[q]));
                __builtin_memcpy(out + (int64_t)chunk * 8, &w, 16);
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) am = max(am, float_to_bits(f[e]) & 0x7fffffffu);
                __builtin_memcpy(out + (int64_t)chunk * 8, f, 32);
            }
        };
        const int n0 = first / 8, n1 = end / 8;  // whole chunks of the output
        for (int i = n0 + tid; i < n1; i += U * kBwdThreads) {
            Chunk<DT> raw[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int chunk = i + u * kBwdThreads;
                if (chunk < n1 && chunk * 8 + 8 <= a.vocab && !nothing) raw[u].load(in + (int64_t)chunk * 8);
                else raw[u].fill();
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int chunk = i + u * kBwdThreads;
                if (chunk >= n1) break;
                float f[8];
                if (nothing) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) f[e] = 0.0f;
                } else {
                    raw[u].widen(f);
                    const bool edge = chunk * 8 + 8 > a.vocab;
                    if (edge)
#pragma unroll
                        for (int e = 0; e < 8; ++e)
                            if (chunk * 8 + e < a.vocab) f[e] = one<DT>(in + (int64_t)chunk * 8 + e);
#pragma unroll
                    for (int e = 0; e < 8; ++e) f[e] = gradient(f[e]);
                    bool look = edge || chunk == t_chunk;
                    if constexpr (TOP) look = look || (marks[(chunk / 32) % kMarks] >> (chunk % 32) & 1u);
                    if (look) special(chunk, f);
                    if (late)
#pragma unroll
                        for (int e = 0; e < 8; ++e) f[e] *= a.inv_t;
                }
                store(chunk, f);
            }
        }
        // the last columns of a row that is no multiple of 8 long
        if (end == a.padded && tid < end % 8) {
            const int col = n1 * 8 + tid;
            float f = 0.0f;
            if (!nothing && col < a.vocab) {
                f = gradient(one<DT>(in + col));
                if (col == (int)target && t_chunk >= 0) f += given;
                if constexpr (TOP)
                    for (int i = 0; i < a.top_k; ++i)
                        if (top_i[i] == col) f = __fmaf_rn(top_d[i], by, f);
                if (late) f *= a.inv_t;
            }
            if constexpr (DT == ODL_BF16) {
                const uint32_t w = pack_bf16x2(f, 0.0f);
                am = max_u16x2(am, abs_bf16x2(w));
                out[col] = (uint16_t)w;
            } else {
                am = max(am, float_to_bits(f) & 0x7fffffffu);
                out[col] = f;
            }
        }
    }
    if (!a.parts) return;
    am = block_max_u32(DT == ODL_BF16 ? fold_u16x2_to_f32bits(am) : am, red);
    if (tid == 0) a.parts[blockIdx.x] = bits_to_float(am);
    if (blockIdx.x == 0)
        for (int j = (int)gridDim.x + tid; j < kParts; j += kBwdThreads) a.parts[j] = 0.0f;
}

int check(const char *who, int dtype, int64_t rows, int64_t stride, int64_t padded, int64_t vocab, int top_k, float inv_t) {
    if (rows < 0 || stride < 0) return set_error(ODL_ERR_ARG, "%s: negative shape", who);
    if (dtype != ODL_BF16 && dtype != ODL_F32) return set_error(ODL_ERR_ARG, "%s: dtype %d", who, dtype);
    if (vocab < 1 || vocab > padded || padded > (1 << 24)) return set_error(ODL_ERR_SHAPE, "%s: %lld of %lld columns (1 to 2^24)", who, (long long)vocab, (long long)padded);
    if (rows >= (1 << 22)) return set_error(ODL_ERR_SHAPE, "%s: %lld rows (up to 2^22 - 1)", who, (long long)rows);   // (lanes of a launch are counted in 32 bits)
    if (top_k < 0 || top_k > kMaxTop || top_k > vocab) return set_error(ODL_ERR_ARG, "%s: top_k %d (0 to %d, and to the vocabulary)", who, top_k, kMaxTop);
    if (!(inv_t >= 0.99e-30f && inv_t <= 1.01e30f)) return set_error(ODL_ERR_ARG, "%s: a temperature from 1e-30 to 1e30", who);
    return ODL_OK;
}

// Blocks that share a row: few rows of a large vocabulary keep a compute unit each busy with their exponentials alone.  us, one block a row / shared,
// no alternatives and 20: 1 x 151936 12.3, 16.9 / 6.2, 12.1; 64 x 128256 10.7, 15.5 / 7.7, 13.9; 100 x 151936 15.4, 20.3 / 12.1, 18.2; 1 x 100352 8.5, 13.2 / 6.0,
// 11.7; 1 x 65536, 32 x 65536 6.3, 11.0 and 6.7, 11.4 / 5.7, 11.6 and 6.4, 12.1, which pays for no second launch.  Parts of 8192: 13.2 to 14.7 for 16.
int parts_of(int64_t rows, int64_t vocab) {
    if (vocab < 98304) return 1;
    int64_t p = device_cu_count() / rows;
    p = p < vocab / 16384 ? p : vocab / 16384;
    return p < 2 ? 1 : p < kMaxParts ? (int)p : kMaxParts;
}

}  // namespace
}  // namespace odl

using namespace odl;

// Floats of the workspace that a call needs; 0: none.
extern "C" int64_t odl_fp8_token_logprobs_workspace(int64_t rows, int64_t vocab, int top_k) {
    if (rows < 1 || rows >= (1 << 22) || vocab < 1 || top_k < 0 || top_k > kMaxTop) return 0;
    const int parts = parts_of(rows, vocab);
    return parts > 1 ? rows * parts * (3 + 2 * top_k) : 0;
}

extern "C" int odl_fp8_token_logprobs(const void *logits, int dtype, int64_t rows, int64_t stride, int64_t vocab, const int64_t *targets,
                                      int64_t ignore_index, float inv_temperature, int top_k, float *logprobs, float *entropy, float *stats,
                                      float *top_logprobs, int64_t *top_ids, float *workspace, int64_t workspace_bytes, odl_stream_t stream_) {
    hipStream_t stream = reinterpret_cast<hipStream_t>(stream_);
    if (const int rc = check("odl_fp8_token_logprobs", dtype, rows, stride, vocab, vocab, top_k, inv_temperature)) return rc;
    if (rows == 0) return ODL_OK;
    if (!logits || !targets || !logprobs || !entropy || (top_k && (!top_logprobs || !top_ids)))
        return set_error(ODL_ERR_ARG, "odl_fp8_token_logprobs: null pointer");
    const int64_t needed = odl_fp8_token_logprobs_workspace(rows, vocab, top_k);
    if (needed && (!workspace || workspace_bytes / 4 < needed))
        return set_error(ODL_ERR_ARG, "odl_fp8_token_logprobs: a workspace of %lld floats is needed", (long long)needed);
    Forward a = {};
    a.logits = logits; a.targets = targets; a.rows = rows; a.stride = stride; a.ignore_index = ignore_index;
    a.vocab = (int)vocab; a.top_k = top_k; a.c = inv_temperature * kLog2e;
    a.logprobs = logprobs; a.entropy = entropy; a.stats = stats; a.top_logprobs = top_logprobs; a.top_ids = top_ids;
    a.parts = needed ? parts_of(rows, vocab) : 1;
    a.span = (int)((vocab + a.parts - 1) / a.parts + 7) / 8 * 8;
    a.partial = workspace;
    if (needed) {
        const dim3 shared((unsigned)rows, (unsigned)a.parts);
        if (dtype == ODL_BF16) {
            hipLaunchKernelGGL((token_logprobs_kernel<ODL_BF16, 512, true>), shared, dim3(512), 0, stream, a);
            hipLaunchKernelGGL(token_logprobs_join_kernel<ODL_BF16>, dim3((unsigned)rows), dim3(256), 0, stream, a);
        } else {
            hipLaunchKernelGGL((token_logprobs_kernel<ODL_F32, 512, true>), shared, dim3(512), 0, stream, a);
            hipLaunchKernelGGL(token_logprobs_join_kernel<ODL_F32>, dim3((unsigned)rows), dim3(256), 0, stream, a);
        }
        return check_launch("odl_fp8_token_logprobs");
    }
    const dim3 grid((unsigned)rows);
    // Lanes of a row's block, us with 256 / 512 / 1024: 8192 x 50257 bf16 160 / 155 / 190, 2048 rows 44.8 / 42.5 / 46.4, 16 x 32000 (top 20) 10.1 / 9.4 / 10.6;
    // short rows, and rows of middle length where there are many, have less to do than a wide block to agree on: 2000 x 1000
    // 11.4 / 17.5 / 30.5, 700 x 32000 15.3 / 17.1 / 20.5; few long ones (top 20): 16 x 81920 - / 12.5 / 12.9
    const int threads = vocab <= 4096 || (vocab <= 40000 && rows >= 512) ? 256 : 512;
#define ODL_LPF(DT, THREADS) hipLaunchKernelGGL((token_logprobs_kernel<DT, THREADS, false>), grid, dim3(THREADS), 0, stream, a)
#define ODL_LPF_DT(THREADS) do { if (dtype == ODL_BF16) ODL_LPF(ODL_BF16, THREADS); else ODL_LPF(ODL_F32, THREADS); } while (0)
    if (threads == 256) ODL_LPF_DT(256);
    else ODL_LPF_DT(512);
#undef ODL_LPF_DT
#undef ODL_LPF
    return check_launch("odl_fp8_token_logprobs");
}

extern "C" int odl_fp8_token_logprobs_bwd(const void *logits, int dtype, int64_t rows, int64_t stride, int64_t vocab, int64_t padded,
                                          const int64_t *targets, int64_t ignore_index, float inv_temperature, int top_k, const int64_t *top_ids,
                                          const float *stats, const float *entropy, const float *d_logprobs, const float *d_entropy,
                                          const float *d_top, void *dlogits, float *parts, odl_stream_t stream_) {
    hipStream_t stream = reinterpret_cast<hipStream_t>(stream_);
    if (const int rc = check("odl_fp8_token_logprobs_bwd", dtype, rows, stride, padded, vocab, top_k, inv_temperature)) return rc;
    if ((rows > 0 && (!logits || !targets || !stats || !entropy || !dlogits)) || (d_top && top_k && !top_ids))
        return set_error(ODL_ERR_ARG, "odl_fp8_token_logprobs_bwd: null pointer");
    Backward a = {};
    a.logits = logits; a.targets = targets; a.top_ids = top_ids; a.d_logprobs = d_logprobs; a.d_entropy = d_entropy; a.d_top = d_top;
    a.stats = stats; a.entropy = entropy; a.rows = rows; a.stride = stride; a.ignore_index = ignore_index;
    a.vocab = (int)vocab; a.padded = (int)padded; a.top_k = d_top ? top_k : 0; a.inv_t = inv_temperature; a.dlogits = dlogits; a.parts = parts;
    const int64_t chunks = (padded + 7) / 8, cap = device_cu_count() * 2 < kParts ? device_cu_count() * 2 : kParts;
    // items of four chunks a lane where there are rows enough, smaller ones where there are few
    int64_t sections = (padded + 4 * 8 * kBwdThreads - 1) / (4 * 8 * kBwdThreads);
    if (rows > 0 && rows * sections < cap) sections = (cap + rows - 1) / rows;
    const int64_t most = (chunks + 63) / 64;                      // (a chunk for every lane of a wave)
    sections = sections < most ? sections : most;
    a.section = (int)((chunks + sections - 1) / sections * 8);
    a.sections = (int)((padded + a.section - 1) / a.section);
    a.items = rows * a.sections;
    const dim3 grid((unsigned)(a.items < 1 ? 1 : a.items < cap ? a.items : cap));
#define ODL_LPB(DT, TOP) hipLaunchKernelGGL((token_logprobs_bwd_kernel<DT, TOP>), grid, dim3(kBwdThreads), 0, stream, a)
    if (dtype == ODL_BF16) { if (a.top_k) ODL_LPB(ODL_BF16, true); else ODL_LPB(ODL_BF16, false); }
    else { if (a.top_k) ODL_LPB(ODL_F32, true); else ODL_LPB(ODL_F32, false); }
#undef ODL_LPB
    return check_launch("odl_fp8_token_logprobs_bwd");
}
