// Verification of drafted tokens.  With p = softmax(x / T) of the model's logits and q that of the drafter's (or all on the drafted token where there are
// none), draft d_j of a sequence is accepted while u_j q_j(d_j) < p_j(d_j).  Behind the first refusal the token is drawn from max(p - q, 0), behind the
// last draft from p: the least i with sum_{k <= i} r_k > u sum_k r_k.  What is emitted is then distributed as the model alone would have it.
//
// Which token it is hangs on sums over the vocabulary next to borders: with n borders and sums that are off by e of their whole, one in 1 / (n e) draws
// would differ.  In fp32 that is one in a hundred for 10^5 tokens; so exponentials and sums are held in 64 bits (2^r by its series to the
// eleventh power, 6e-15), which the vector units do at the rate that memory delivers: some 20 operations an element.
//
// Three launches.  The first reads every row once, in parts, and leaves a maximum and a sum of each.  In the second every sequence has a block for each
// part of a row: each works out for itself which draft is the first to be refused and sums what is left of its part of that row (again from
// memory: one row of each sequence).  In the third a block a sequence finds the part that holds the number drawn and the token in it.
// T = 0: p is all on the largest logit, the lowest of them, and the second launch ends it.
//
// One launch for both of the first two would need the blocks of a row to wait for each other; tickets for the last block of a row to go on took longer than the launch
// that they save.  Measured (calls in a row): 17 us for one sequence of 3 rows, 37 for 24 of 108 rows in all (50257 columns of bf16), which is the three launches' latency
// (their bytes take 4), 149 for 64 of 6 rows (151936 of fp32), of which 84 are bytes: the first launch runs at 4.2 TB/s, the second reads one row of each side again.
#include "common.h"

#pragma clang fp contract(off)

namespace odl {
namespace {

constexpr int kThreads = 256, kPiece = kThreads * 8;           // elements that a block reads at a time
constexpr int kMaxParts = 128;

struct Part {                                    // of a part of a row: its maximum, the sum against it, the lowest place of the maximum
    double s;
    float m;
    int at;
};

struct Verify {
    const void *logits, *drafts;
    int64_t stride, draft_stride;
    const int64_t *tokens;
    const int32_t *offsets;
    const float *uniforms;
    int rows, seqs, vocab, parts, span;          // parts of a row, columns of one (a multiple of kPiece)
    double c;                                    // log2(e) / T
    int32_t *accepted;
    int64_t *out;
    float *logprobs;
    Part *part;                                  // [2][rows][parts]
    double *left;                                // [seqs][parts]
    struct Stop *stop;                           // [seqs]
};

// 2^t
__device__ __forceinline__ double power(double t) {
    t = fmax(t, -2000.0);
    const double n = __builtin_rint(t), r = t - n;
    double p = 4.4455382718708114976e-10;
    p = __builtin_fma(p, r, 7.0549116208011233299e-9);
    p = __builtin_fma(p, r, 1.0178086009239699728e-7);
    p = __builtin_fma(p, r, 1.3215486790144309488e-6);
    p = __builtin_fma(p, r, 1.5252733804059840280e-5);
    p = __builtin_fma(p, r, 1.5403530393381609954e-4);
    p = __builtin_fma(p, r, 1.3333558146428443423e-3);
    p = __builtin_fma(p, r, 9.6181291076284771620e-3);
    p = __builtin_fma(p, r, 5.5504108664821579953e-2);
    p = __builtin_fma(p, r, 2.4022650695910071233e-1);
    p = __builtin_fma(p, r, 6.9314718055994530942e-1);
    p = __builtin_fma(p, r, 1.0);
    return __builtin_ldexp(p, (int)n);
}
__device__ __forceinline__ double weight(float x, float m, double c) { return power(((double)x - (double)m) * c); }

template <int DT>
__device__ __forceinline__ float element(const void *row, int64_t i) {
    if constexpr (DT == ODL_BF16) return bits_to_float((uint32_t) reinterpret_cast<const uint16_t *>(row)[i] << 16);
    else return reinterpret_cast<const float *>(row)[i];
}
// eight elements from column i on, at any alignment; -inf behind the end
template <int DT>
__device__ __forceinline__ void load8(const void *row, int i, int end, float (&f)[8]) {
    if (i + 8 <= end) {
        if constexpr (DT == ODL_BF16) {
            uint32_t w[4];
            __builtin_memcpy(w, reinterpret_cast<const uint16_t *>(row) + i, sizeof(w));
#pragma unroll
            for (int k = 0; k < 4; ++k) { f[2 * k] = bf16_lo(w[k]); f[2 * k + 1] = bf16_hi(w[k]); }
        } else {
            __builtin_memcpy(f, reinterpret_cast<const float *>(row) + i, sizeof(f));
        }
    } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) f[k] = i + k < end ? element<DT>(row, i + k) : -INFINITY;
    }
}
template <int DT>
__device__ __forceinline__ const void *row_at(const void *base, int64_t row, int64_t stride) {
    return static_cast<const uint8_t *>(base) + row * stride * (DT == ODL_BF16 ? 2 : 4);
}

// A value of another lane of a row of 16 (a DPP control word), and over the wave what F makes of all lanes' values, in every lane.
template <int CTRL, class T>
__device__ __forceinline__ T from_dpp(T v) {
    uint32_t w[sizeof(T) / 4];
    __builtin_memcpy(w, &v, sizeof(T));
#pragma unroll
    for (int i = 0; i < (int)(sizeof(T) / 4); ++i) w[i] = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)w[i], CTRL, 0xf, 0xf, false);
    __builtin_memcpy(&v, w, sizeof(T));
    return v;
}
template <class T, class F>
__device__ __forceinline__ T over_wave(T v, F f) {
    v = f(v, from_dpp<0xB1>(v));                 // lane ^ 1, ^ 2, the other quad of 8, the other half of 16
    v = f(v, from_dpp<0x4E>(v));
    v = f(v, from_dpp<0x141>(v));
    v = f(v, from_dpp<0x140>(v));
    uint32_t w[sizeof(T) / 4], a[sizeof(T) / 4], b[sizeof(T) / 4];
    T x, y;
    __builtin_memcpy(w, &v, sizeof(T));
#pragma unroll
    for (int i = 0; i < (int)(sizeof(T) / 4); ++i) {
        const auto r = __builtin_amdgcn_permlane16_swap(w[i], w[i], false, false);
        a[i] = r[0], b[i] = r[1];
    }
    __builtin_memcpy(&x, a, sizeof(T));
    __builtin_memcpy(&y, b, sizeof(T));
    v = f(x, y);
    __builtin_memcpy(w, &v, sizeof(T));
#pragma unroll
    for (int i = 0; i < (int)(sizeof(T) / 4); ++i) {
        const auto r = __builtin_amdgcn_permlane32_swap(w[i], w[i], false, false);
        a[i] = r[0], b[i] = r[1];
    }
    __builtin_memcpy(&x, a, sizeof(T));
    __builtin_memcpy(&y, b, sizeof(T));
    return f(x, y);
}
__device__ __forceinline__ double wave_sum(double v) { return over_wave(v, [](double a, double b) { return a + b; }); }
__device__ __forceinline__ float wave_max(float v) { return over_wave(v, [](float a, float b) { return fmaxf(a, b); }); }
__device__ __forceinline__ int wave_min(int v) { return over_wave(v, [](int a, int b) { return min(a, b); }); }

// The parts of a wave's lanes as one, in every lane.  (Sums of NaN rows stay NaN.)
template <bool GREEDY>
__device__ __forceinline__ Part wave_join(const Part &a, double c) {
    Part r = {a.s, wave_max(a.m), INT32_MAX};
    if (r.m != -INFINITY) r.s = a.m == r.m ? a.s : a.s * weight(a.m, r.m, c);
    r.s = wave_sum(r.s);
    if (GREEDY) r.at = wave_min(a.m == r.m ? a.at : INT32_MAX);
    return r;
}

// The sequence of a row: how many of them end at or in front of it.
__device__ __forceinline__ int sequence_of(const int32_t *offsets, int seqs, int row) {
    const int lane = threadIdx.x % kWave;
    int s = 0;
    for (int s0 = 0; s0 < seqs; s0 += kWave) s += __popcll(__ballot(s0 + lane < seqs && offsets[s0 + lane + 1] <= row));
    return __builtin_amdgcn_readfirstlane(s);
}

template <int DT, bool GREEDY>
__global__ __launch_bounds__(kThreads) void draft_sums_kernel(Verify a) {
    __shared__ Part waves[kThreads / kWave];
    const int row = blockIdx.y, part = blockIdx.x, side = blockIdx.z, tid = threadIdx.x;
    if (side == 0 && part == 0 && tid == 0) {
        a.out[row] = -1;
        a.logprobs[row] = 0.0f;
    }
    const int s = sequence_of(a.offsets, a.seqs, row);
    if (s >= a.seqs || (side == 1 && a.offsets[s + 1] == row + 1)) return;               // (nobody reads the drafter's answer to the last token)
    const void *x = side ? row_at<DT>(a.drafts, row, a.draft_stride) : row_at<DT>(a.logits, row, a.stride);
    const int begin = part * a.span, end = min(begin + a.span, a.vocab);
    Part mine = {0.0, -INFINITY, INT32_MAX};
    bool odd = false;
    for (int base = begin; base < end; base += 4 * kPiece) {
        float f[4][8];
#pragma unroll
        for (int k = 0; k < 4; ++k) load8<DT>(x, base + k * kPiece + tid * 8, end, f[k]);
        float m = -INFINITY;
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                m = fmaxf(m, f[k][i]);
                odd |= !(f[k][i] < INFINITY);
            }
        if (m == -INFINITY) continue;
        if constexpr (GREEDY) {
            if (m > mine.m) {
                int at = INT32_MAX;
#pragma unroll
                for (int k = 3; k >= 0; --k)
#pragma unroll
                    for (int i = 7; i >= 0; --i) at = f[k][i] == m ? base + k * kPiece + tid * 8 + i : at;
                mine.at = at;
            }
        }
        if (m > mine.m) {
            mine.s = mine.m == -INFINITY ? 0.0 : mine.s * weight(mine.m, m, a.c);
            mine.m = m;
        }
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (base + k * kPiece < end) {
#pragma unroll
                for (int i = 0; i < 8; ++i) mine.s += weight(f[k][i], mine.m, a.c);
            }
    }
    if (odd) mine.s = __builtin_nan("");
    mine = wave_join<GREEDY>(mine, a.c);
    if (tid % kWave == 0) waves[tid / kWave] = mine;
    __syncthreads();
    if (tid >= kWave) return;
    mine = {0.0, -INFINITY, INT32_MAX};
    if (tid < kThreads / kWave) mine = waves[tid];
    mine = wave_join<GREEDY>(mine, a.c);
    if (tid == 0) a.part[((int64_t)side * a.rows + row) * a.parts + part] = mine;
}

// A row's parts as one, in every lane of a wave: the loads, and what they make.
struct Parts {
    Part p[kMaxParts / kWave];
    __device__ __forceinline__ void load(const Verify &a, int side, int row) {
        const Part *from = a.part + ((int64_t)side * a.rows + row) * a.parts;
        const int lane = threadIdx.x % kWave;
#pragma unroll
        for (int i = 0; i < kMaxParts / kWave; ++i) {
            p[i] = {0.0, -INFINITY, INT32_MAX};
            if (lane + i * kWave < a.parts) p[i] = from[lane + i * kWave];
        }
    }
    template <bool GREEDY>
    __device__ __forceinline__ Part whole(const Verify &a) const {
        Part r = p[0];
#pragma unroll
        for (int i = 1; i < kMaxParts / kWave; ++i)
            if (a.parts > i * kWave) {
                const float top = fmaxf(r.m, p[i].m);
                if (top != -INFINITY) r.s = (r.m == top ? r.s : r.s * weight(r.m, top, a.c)) + (p[i].m == top ? p[i].s : p[i].s * weight(p[i].m, top, a.c));
                else r.s += p[i].s;
                if (GREEDY) r.at = r.m == p[i].m ? min(r.at, p[i].at) : r.m > p[i].m ? r.at : p[i].at;
                r.m = top;
            }
        return wave_join<GREEDY>(r, a.c);
    }
};

__device__ __forceinline__ bool sound(const Part &p) { return p.s > 0.0 && p.s < INFINITY; }

struct Row {                                     // a distribution: the maximum of its logits, and 1 / sum
    float m;
    double by;
};
struct Stop {                                    // where a sequence stops and what is drawn from there
    Row p, q;
    int row, draft;                              // draft: what is to be taken off p as a whole, -1 where nothing is
    int residual, number;                        // residual: max(p - q, 0) and not p; number: the row whose number draws, -1: the answer is there
};

// What is left of a lane's eight elements of each of four pieces from column `base` on (32 columns a lane in all, loaded at once): f(piece, element, it).
template <int DT, class F>
__device__ __forceinline__ void left32(const Verify &a, const Stop &st, int base, int end, F f) {
    const void *p = row_at<DT>(a.logits, st.row, a.stride), *q = row_at<DT>(a.drafts, st.row, a.draft_stride);
    float x[4][8], y[4][8];
#pragma unroll
    for (int k = 0; k < 4; ++k) load8<DT>(p, base + k * kPiece + threadIdx.x * 8, end, x[k]);
    if (st.residual)
#pragma unroll
        for (int k = 0; k < 4; ++k) load8<DT>(q, base + k * kPiece + threadIdx.x * 8, end, y[k]);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const int at = base + k * kPiece;
        if (at >= end) break;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            double r = weight(x[k][i], st.p.m, a.c) * st.p.by;
            if (st.residual) r = fmax(r - weight(y[k][i], st.q.m, a.c) * st.q.by, 0.0);
            if (at + (int)threadIdx.x * 8 + i == st.draft) r = 0.0;
            f(k, i, r);
        }
    }
}

// How far a sequence's drafts hold, and what is left of a part of the row behind which it stops.
template <int DT, bool GREEDY>
__global__ __launch_bounds__(kThreads) void draft_stop_kernel(Verify a) {
    constexpr int kWaves = kThreads / kWave, kBoth = 2;        // rows a wave looks at at a time
    __shared__ Stop stop;
    __shared__ bool agreed[kBoth * kWaves];
    __shared__ Part found[kBoth * kWaves][2];
    __shared__ double sums[kWaves];
    const int s = blockIdx.y, part = blockIdx.x, tid = threadIdx.x, wave = tid / kWave, lane = tid % kWave;
    const int first = min(max(a.offsets[s], 0), a.rows), n = min(a.offsets[s + 1], a.rows) - first;
    if (n <= 0) {
        if (part == 0 && tid == 0) {
            a.accepted[s] = 0;
            a.stop[s].number = -1;
        }
        return;
    }
    for (int at = 0;; at += kBoth * kWaves) {
        Parts of_row[kBoth], of_draft[kBoth];
        int64_t draft[kBoth];
        float x[kBoth], y[kBoth], logprob[kBoth];
#pragma unroll
        for (int b = 0; b < kBoth; ++b) {
            const int j = at + b * kWaves + wave, row = first + j;
            draft[b] = j < n - 1 ? a.tokens[row + 1] : -1;
            if (j < n) of_row[b].load(a, 0, row);
            if (!GREEDY && a.drafts && j < n - 1) of_draft[b].load(a, 1, row);
            if (draft[b] >= a.vocab) draft[b] = -1;
        }
#pragma unroll
        for (int b = 0; b < kBoth; ++b) {
            const int row = first + at + b * kWaves + wave;
            if (draft[b] < 0) continue;
            x[b] = element<DT>(row_at<DT>(a.logits, row, a.stride), draft[b]);
            if (!GREEDY && a.drafts) y[b] = element<DT>(row_at<DT>(a.drafts, row, a.draft_stride), draft[b]);
        }
#pragma unroll
        for (int b = 0; b < kBoth; ++b) {
            const int j = at + b * kWaves + wave, row = first + j;
            bool yes = false;
            if (j < n) {
                const Part p = of_row[b].template whole<GREEDY>(a);
                Part q = {0.0, 0.0f, 0};
                if (!GREEDY && a.drafts && j < n - 1) q = of_draft[b].template whole<GREEDY>(a);
                if (draft[b] >= 0 && sound(p)) {
                    if (GREEDY) yes = draft[b] == p.at;
                    else yes = (double)a.uniforms[row] * (a.drafts ? weight(y[b], q.m, a.c) / q.s : 1.0) < weight(x[b], p.m, a.c) / p.s;
                    if (yes && part == 0) logprob[b] = (float)(((double)x[b] - (double)p.m) * a.c * 0.69314718055994530942 - log(p.s));
                }
                if (lane == 0) found[b * kWaves + wave][0] = p, found[b * kWaves + wave][1] = q;
            }
            if (lane == 0) agreed[b * kWaves + wave] = yes;
        }
        __syncthreads();
        int w = 0;
        while (w < kBoth * kWaves && agreed[w]) ++w;
#pragma unroll
        for (int b = 0; b < kBoth; ++b)
            if (part == 0 && lane == 0 && b * kWaves + wave < w) {
                const int row = first + at + b * kWaves + wave;
                a.out[row] = draft[b];
                a.logprobs[row] = logprob[b];
            }
        if (w < kBoth * kWaves) {
            if (tid == 0) {
                const Part p = found[w][0], q = found[w][1];
                const int j = at + w, row = first + j;
                const int64_t d = j < n - 1 ? a.tokens[row + 1] : -1;
                stop.row = row;
                stop.draft = d >= 0 && d < a.vocab && !a.drafts ? (int)d : -1;
                stop.p = {p.m, 1.0 / p.s};
                stop.q = {q.m, 1.0 / q.s};
                stop.residual = j < n - 1 && a.drafts && sound(q);
                stop.number = GREEDY || !sound(p) ? -1 : first + n - 1;
                if (part == 0) {
                    a.accepted[s] = j;
                    if (GREEDY || !sound(p)) {
                        a.out[row] = sound(p) ? p.at : -1;
                        a.logprobs[row] = sound(p) ? (float)-log(p.s) : __builtin_nanf("");
                    }
                    a.stop[s] = stop;
                }
            }
            break;
        }
        __syncthreads();
    }
    __syncthreads();
    if (GREEDY || stop.number < 0) return;
    const Stop st = stop;
    double sum = 0.0;
    if (!st.residual && st.draft < 0) {          // p as it is: summed already
        if (tid == 0) {
            const Part p = a.part[(int64_t)st.row * a.parts + part];
            a.left[(int64_t)s * a.parts + part] = p.m == -INFINITY ? 0.0 : p.s * weight(p.m, st.p.m, a.c) * st.p.by;
        }
        return;
    }
    const int begin = part * a.span, end = min(begin + a.span, a.vocab);
    for (int base = begin; base < end; base += 4 * kPiece) left32<DT>(a, st, base, end, [&](int, int, double r) { sum += r; });
    sum = wave_sum(sum);
    if (lane == 0) sums[wave] = sum;
    __syncthreads();
    if (tid == 0) a.left[(int64_t)s * a.parts + part] = (sums[0] + sums[1]) + (sums[2] + sums[3]);
}

// The part that holds the number drawn, and the token in it.
template <int DT>
__global__ __launch_bounds__(kThreads) void draft_pick_kernel(Verify a) {
    constexpr int kWaves = kThreads / kWave;
    __shared__ double sums[kWaves][4], lefts[kMaxParts];
    __shared__ int hits[kWaves];
    const int s = blockIdx.x, tid = threadIdx.x, wave = tid / kWave, lane = tid % kWave;
    Stop st = a.stop[s];
    for (int i = tid; i < a.parts; i += kThreads) lefts[i] = a.left[(int64_t)s * a.parts + i];
    if (st.number < 0) return;                   // (what else the workspace holds of this sequence is of no call)
    const double u = a.uniforms[st.number];
    __syncthreads();
    double total = 0.0;
    for (int i = 0; i < a.parts; ++i) total += lefts[i];
    if (!(total > 0.0)) {                        // nothing is left (p and q are the same): p itself
        st.residual = 0;
        st.draft = -1;
        __syncthreads();
        for (int i = tid; i < a.parts; i += kThreads) {
            const Part p = a.part[(int64_t)st.row * a.parts + i];
            lefts[i] = p.m == -INFINITY ? 0.0 : p.s * weight(p.m, st.p.m, a.c) * st.p.by;
        }
        __syncthreads();
        total = 0.0;
        for (int i = 0; i < a.parts; ++i) total += lefts[i];
    }
    const double want = u * total;
    double before = 0.0;
    int in = -1, some = 0;
    for (int i = 0; i < a.parts && in < 0; ++i) {
        if (lefts[i] > 0.0) some = i;
        if (before + lefts[i] > want) in = i;
        else before += lefts[i];
    }
    if (in < 0) {                                // (a number of 1 or more, or sums that end a last place short: the last token that there is)
        in = some;
        before -= lefts[some];
    }
    const int from = in * a.span, to = min(from + a.span, a.vocab);
    int hit = INT32_MAX, tail = -1;              // the token, and the last that has any weight
    for (int base = from; base < to && hit == INT32_MAX; base += 4 * kPiece) {
        double r[4][8], local[4] = {0.0, 0.0, 0.0, 0.0}, upto[4];
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
            for (int i = 0; i < 8; ++i) r[k][i] = 0.0;
        left32<DT>(a, st, base, to, [&](int k, int i, double v) {
            r[k][i] = v;
            local[k] += v;
            if (v > 0.0) tail = base + k * kPiece + tid * 8 + i;
        });
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            upto[k] = local[k];
#pragma unroll
            for (int off = 1; off < kWave; off <<= 1) {
                const double v = __shfl_up(upto[k], off, kWave);
                if (lane >= off) upto[k] += v;
            }
        }
        __syncthreads();
        if (lane == kWave - 1)
#pragma unroll
            for (int k = 0; k < 4; ++k) sums[wave][k] = upto[k];
        __syncthreads();
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            double c = before + (upto[k] - local[k]);
            for (int w = 0; w < wave; ++w) c += sums[w][k];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                c += r[k][i];
                if (c > want && r[k][i] > 0.0) hit = min(hit, base + k * kPiece + tid * 8 + i);
            }
            before += (sums[0][k] + sums[1][k]) + (sums[2][k] + sums[3][k]);
        }
        hit = wave_min(hit);
        if (lane == 0) hits[wave] = hit;
        __syncthreads();
        hit = min(min(hits[0], hits[1]), min(hits[2], hits[3]));
    }
    if (hit == INT32_MAX) {                      // (uniform)
        tail = -wave_min(-tail);
        __syncthreads();
        if (lane == 0) hits[wave] = tail;
        __syncthreads();
        hit = max(max(hits[0], hits[1]), max(hits[2], hits[3]));
    }
    if (tid == 0) {
        a.out[st.row] = hit;
        const float x = element<DT>(row_at<DT>(a.logits, st.row, a.stride), max(hit, 0));
        a.logprobs[st.row] = (float)(((double)x - (double)st.p.m) * a.c * 0.69314718055994530942 + log(st.p.by));
    }
}

// Parts of a row: of 8192 columns where that makes two blocks a compute unit, else of 2048.
int parts_of(int64_t rows, int64_t vocab, int &span) {
    span = rows * ((vocab + 4 * kPiece - 1) / (4 * kPiece)) >= 2 * (int64_t)device_cu_count() ? 4 * kPiece : kPiece;
    if ((vocab + span - 1) / span > kMaxParts) span = (int)(((vocab + kMaxParts - 1) / kMaxParts + kPiece - 1) / kPiece * kPiece);
    return (int)((vocab + span - 1) / span);
}

int check(const char *who, int64_t rows, int64_t seqs, int64_t vocab) {
    if (rows < 0 || seqs < 0) return set_error(ODL_ERR_ARG, "%s: negative shape", who);
    if (vocab < 1 || vocab > 1 << 24) return set_error(ODL_ERR_SHAPE, "%s: a vocabulary of %lld (1 to 2^24)", who, (long long)vocab);
    if (rows > 65535 || seqs > 65535) return set_error(ODL_ERR_SHAPE, "%s: up to 65535 rows and sequences", who);
    return ODL_OK;
}

}  // namespace
}  // namespace odl

using namespace odl;

extern "C" int64_t odl_fp8_verify_drafts_workspace(int64_t rows, int64_t seqs, int64_t vocab) {
    if (check("odl_fp8_verify_drafts_workspace", rows, seqs, vocab)) return -1;
    int span;
    const int64_t parts = parts_of(rows, vocab, span);
    return (rows * 2 * parts * (int64_t)sizeof(Part) + seqs * (int64_t)(sizeof(Stop) + parts * sizeof(double))) / 4;
}

extern "C" int odl_fp8_verify_drafts(const void *logits, int64_t stride, const void *draft_logits, int64_t draft_stride, int dtype, int64_t rows, int64_t vocab,
                                     const int64_t *tokens, const int32_t *offsets, int64_t seqs, const float *uniforms, double temperature, int32_t *accepted,
                                     int64_t *out_tokens, float *logprobs, float *workspace, int64_t workspace_floats, odl_stream_t stream_) {
    static const char who[] = "odl_fp8_verify_drafts";
    if (const int rc = check(who, rows, seqs, vocab)) return rc;
    if (dtype != ODL_BF16 && dtype != ODL_F32) return set_error(ODL_ERR_ARG, "%s: dtype %d", who, dtype);
    if (!(temperature == 0.0 || (temperature >= 1e-30 && temperature <= 1e30))) return set_error(ODL_ERR_ARG, "%s: temperature %g (0, or 1e-30 to 1e30)", who, temperature);
    if (!offsets || (seqs > 0 && !accepted) || (rows > 0 && (!logits || !tokens || !uniforms || !out_tokens || !logprobs))) return set_error(ODL_ERR_ARG, "%s: null pointer", who);
    if (stride < 0 || draft_stride < 0) return set_error(ODL_ERR_ARG, "%s: negative stride", who);
    const int64_t need = odl_fp8_verify_drafts_workspace(rows, seqs, vocab);
    if (need > 0 && (!workspace || workspace_floats < need || (reinterpret_cast<uintptr_t>(workspace) & 15)))
        return set_error(ODL_ERR_ARG, "%s: a workspace of %lld floats, 16-byte aligned", who, (long long)need);
    Verify a;
    const bool greedy = temperature == 0.0;
    a.logits = logits, a.drafts = greedy ? nullptr : draft_logits, a.stride = stride, a.draft_stride = draft_stride;
    a.tokens = tokens, a.offsets = offsets, a.uniforms = uniforms;
    a.rows = (int)rows, a.seqs = (int)seqs, a.vocab = (int)vocab;
    a.parts = parts_of(rows, vocab, a.span);
    a.c = 1.4426950408889634074 / (greedy ? 1.0 : temperature);
    a.accepted = accepted, a.out = out_tokens, a.logprobs = logprobs;
    a.part = reinterpret_cast<Part *>(workspace);
    a.stop = reinterpret_cast<Stop *>(a.part + 2 * rows * a.parts);
    a.left = reinterpret_cast<double *>(a.stop + seqs);
    hipStream_t stream = reinterpret_cast<hipStream_t>(stream_);
#define ODL_VERIFY(KERNEL, GRID)                                                                                              \
    do {                                                                                                                      \
        if (dtype == ODL_BF16 && greedy) hipLaunchKernelGGL((KERNEL<ODL_BF16, true>), GRID, dim3(kThreads), 0, stream, a);    \
        else if (dtype == ODL_BF16) hipLaunchKernelGGL((KERNEL<ODL_BF16, false>), GRID, dim3(kThreads), 0, stream, a);        \
        else if (greedy) hipLaunchKernelGGL((KERNEL<ODL_F32, true>), GRID, dim3(kThreads), 0, stream, a);                     \
        else hipLaunchKernelGGL((KERNEL<ODL_F32, false>), GRID, dim3(kThreads), 0, stream, a);                                \
    } while (0)
    if (rows > 0) ODL_VERIFY(draft_sums_kernel, dim3((unsigned)a.parts, (unsigned)rows, a.drafts ? 2u : 1u));
    if (seqs > 0) ODL_VERIFY(draft_stop_kernel, dim3(greedy || rows == 0 ? 1u : (unsigned)a.parts, (unsigned)seqs));
#undef ODL_VERIFY
    if (seqs > 0 && rows > 0 && !greedy) {
        if (dtype == ODL_BF16) hipLaunchKernelGGL((draft_pick_kernel<ODL_BF16>), dim3((unsigned)seqs), dim3(kThreads), 0, stream, a);
        else hipLaunchKernelGGL((draft_pick_kernel<ODL_F32>), dim3((unsigned)seqs), dim3(kThreads), 0, stream, a);
    }
    return check_launch(who);
}
