// Verification of drafted tokens.  With p = softmax(x / T) of the model's logits and q that of the drafter's (or all on the drafted token where there are
// none), draft d_j of a sequence is accepted while u_j q_j(d_j) < p_j(d_j).  Behind the first refusal the token is drawn from max(p - q, 0), behind the
// last draft from p: the least i with sum_{k <= i} r_k > u sum_k r_k.  What is emitted is then distributed as the model alone would have it.
//
// Which token it is hangs on sums over the vocabulary next to borders: with n borders and sums that are off by e of their whole, one in 1 / (n e) draws
// would differ.  In fp32 that is one in a hundred for 10^5 tokens; so exponentials and sums are held in 64 bits (2^r by its series to the
// eleventh power, 6e-15), which the vector units do at the rate that memory delivers: some 20 operations an element.
//
// Two launches.  The first reads every row once, in parts, and leaves a maximum and a sum of each.  In the second every sequence has a block for each part of a
// row: each works out for itself which draft is the first to be refused, sums what is left of its part of that row (again from memory: one row
// of each sequence), and the last to arrive finds the part and the token in it.  T = 0: p is all on the largest logit, the lowest of them.
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
    uint32_t *arrived;                           // [seqs]
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

// One of two parts as one.
__device__ __forceinline__ void join(Part &a, double s, float m, int at, double c) {
    const float top = fmaxf(a.m, m);
    if (top == -INFINITY) { a.s += s; return; }                 // (sums of NaN rows stay NaN)
    a.at = a.m == m ? min(a.at, at) : a.m > m ? a.at : at;
    a.s = (a.m == top ? a.s : a.s * weight(a.m, top, c)) + (m == top ? s : s * weight(m, top, c));
    a.m = top;
}
__device__ __forceinline__ void wave_join(Part &a, double c) {
#pragma unroll
    for (int off = kWave / 2; off > 0; off >>= 1) {
        const double s = __shfl_xor(a.s, off, kWave);
        const float m = __shfl_xor(a.m, off, kWave);
        const int at = __shfl_xor(a.at, off, kWave);
        join(a, s, m, at, c);
    }
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
    if (side == 0 && part == 0) {
        if (tid == 0) { a.out[row] = -1; a.logprobs[row] = 0.0f; }
        for (int s = row * kThreads + tid; s < a.seqs; s += a.rows * kThreads) a.arrived[s] = 0;
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
    wave_join(mine, a.c);
    if (tid % kWave == 0) waves[tid / kWave] = mine;
    __syncthreads();
    if (tid) return;
    for (int w = 1; w < kThreads / kWave; ++w) join(mine, waves[w].s, waves[w].m, waves[w].at, a.c);
    a.part[((int64_t)side * a.rows + row) * a.parts + part] = mine;
}

// A row's parts as one, in every lane of a wave.
__device__ __forceinline__ Part whole(const Verify &a, int side, int row) {
    const Part *p = a.part + ((int64_t)side * a.rows + row) * a.parts;
    const int lane = threadIdx.x % kWave;
    Part r = {0.0, -INFINITY, INT32_MAX};
    for (int i = lane; i < a.parts; i += kWave) join(r, p[i].s, p[i].m, p[i].at, a.c);
    wave_join(r, a.c);
    return r;
}

struct Row {                                     // a distribution: the maximum of its logits, and 1 / sum
    float m;
    double by;
};
struct Stop {                                    // where a sequence stops and what is drawn from there
    int row, draft;                              // draft: what the drafter had there, -1 where there is none to take off
    Row p, q;
    int residual;                                // 0: p, 1: p without the draft, 2: max(p - q, 0)
};

__device__ __forceinline__ bool sound(const Part &p) { return p.s > 0.0 && p.s < INFINITY; }

// What is left of eight elements.
template <int DT>
__device__ __forceinline__ void left8(const Verify &a, const Stop &st, int residual, int i, int end, double (&r)[8]) {
    float x[8], y[8];
    load8<DT>(row_at<DT>(a.logits, st.row, a.stride), i, end, x);
    if (residual == 2) load8<DT>(row_at<DT>(a.drafts, st.row, a.draft_stride), i, end, y);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        r[k] = i + k < end ? weight(x[k], st.p.m, a.c) * st.p.by : 0.0;
        if (residual == 2) r[k] = i + k < end ? fmax(r[k] - weight(y[k], st.q.m, a.c) * st.q.by, 0.0) : 0.0;
        if (residual == 1 && i + k == st.draft) r[k] = 0.0;
    }
}

__device__ __forceinline__ double block_sum(double v, double *lds) {
#pragma unroll
    for (int off = kWave / 2; off > 0; off >>= 1) v += __shfl_xor(v, off, kWave);
    __syncthreads();
    if (threadIdx.x % kWave == 0) lds[threadIdx.x / kWave] = v;
    __syncthreads();
    double s = lds[0];
#pragma unroll
    for (int w = 1; w < kThreads / kWave; ++w) s += lds[w];
    return s;
}

template <int DT, bool GREEDY>
__global__ __launch_bounds__(kThreads) void draft_verify_kernel(Verify a) {
    __shared__ Stop stop;
    __shared__ int best, agreed[kThreads / kWave], chosen, last_one;
    __shared__ Part found[kThreads / kWave][2];
    __shared__ double sums[kThreads / kWave], lefts[kMaxParts];
    const int s = blockIdx.y, part = blockIdx.x, tid = threadIdx.x, wave = tid / kWave, lane = tid % kWave;
    const int first = min(max(a.offsets[s], 0), a.rows), n = min(a.offsets[s + 1], a.rows) - first;
    if (n <= 0) {
        if (part == 0 && tid == 0) a.accepted[s] = 0;
        return;
    }
    // how far the drafts are accepted: a wave a row
    int at = 0;
    for (;; at += kThreads / kWave) {
        const int j = at + wave, row = first + j;
        bool yes = false;
        int64_t draft = -1;
        float logprob = 0.0f;
        if (j < n) {
            const Part p = whole(a, 0, row);
            Part q = {0.0, 0.0f, 0};
            if (j < n - 1) {
                const int64_t d = a.tokens[row + 1];
                const bool known = d >= 0 && d < a.vocab;
                if (GREEDY) {
                    yes = sound(p) && d == p.at;
                } else {
                    const float x = known ? element<DT>(row_at<DT>(a.logits, row, a.stride), d) : -INFINITY;
                    const double of_p = known ? weight(x, p.m, a.c) / p.s : 0.0;
                    double of_q = 1.0;
                    if (a.drafts) {
                        q = whole(a, 1, row);
                        of_q = known ? weight(element<DT>(row_at<DT>(a.drafts, row, a.draft_stride), d), q.m, a.c) / q.s : 1.0;
                    }
                    yes = sound(p) && (double)a.uniforms[row] * of_q < of_p;
                }
                if (yes && part == 0) {
                    draft = d;
                    logprob = (float)(((double)element<DT>(row_at<DT>(a.logits, row, a.stride), d) - (double)p.m) * a.c * 0.69314718055994530942 - log(p.s));
                }
            }
            if (lane == 0) found[wave][0] = p, found[wave][1] = q;
        }
        if (lane == 0) agreed[wave] = yes;
        __syncthreads();
        int w = 0;
        while (w < kThreads / kWave && agreed[w]) ++w;
        if (part == 0 && lane == 0 && wave < w) {
            a.out[row] = draft;
            a.logprobs[row] = logprob;
        }
        if (w < kThreads / kWave) {
            at += w;
            if (tid == 0) {
                const Part p = found[w][0], q = found[w][1];
                const int row = first + at;
                const int64_t d = at < n - 1 ? a.tokens[row + 1] : -1;
                stop.row = row;
                stop.draft = d >= 0 && d < a.vocab ? (int)d : -1;
                stop.p = {p.m, 1.0 / p.s};
                stop.q = {q.m, 1.0 / q.s};
                stop.residual = at == n - 1 ? 0 : !a.drafts ? 1 : sound(q) ? 2 : 0;
                best = sound(p) ? p.at : -1;
                if (!sound(p)) stop.residual = -1;
            }
            break;
        }
        __syncthreads();
    }
    __syncthreads();
    const Stop st = stop;
    const double *mine = a.left + (int64_t)s * a.parts;
    if (GREEDY || st.residual < 0) {
        if (part == 0 && tid == 0) {
            a.accepted[s] = at;
            a.out[st.row] = best;
            a.logprobs[st.row] = best < 0 ? __builtin_nanf("") : (float)log(st.p.by);
        }
        return;
    }
    // what is left of this part of the row
    const int begin = part * a.span, end = min(begin + a.span, a.vocab);
    double sum = 0.0;
    if (st.residual == 0) {
        const Part p = a.part[(int64_t)st.row * a.parts + part];
        sum = p.m == -INFINITY ? 0.0 : p.s * weight(p.m, st.p.m, a.c) * st.p.by;
    } else {
        for (int i = begin + tid * 8; i < end; i += kPiece) {
            double r[8];
            left8<DT>(a, st, st.residual, i, end, r);
#pragma unroll
            for (int k = 0; k < 8; ++k) sum += r[k];
        }
        sum = block_sum(sum, sums);
    }
    if (tid == 0) {
        a.left[(int64_t)s * a.parts + part] = sum;
        __threadfence();
        last_one = atomicAdd(a.arrived + s, 1u) == (uint32_t)a.parts - 1;
        __threadfence();
    }
    __syncthreads();
    if (!last_one) return;
    // the last block of the sequence: the part that holds the number drawn, and the token in it
    for (int i = tid; i < a.parts; i += kThreads) lefts[i] = __hip_atomic_load(mine + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    int residual = st.residual;
    double total = 0.0;
    for (int i = 0; i < a.parts; ++i) total += lefts[i];
    if (!(total > 0.0)) {                        // nothing is left (p and q are the same): p itself
        residual = 0;
        __syncthreads();
        for (int i = tid; i < a.parts; i += kThreads) {
            const Part p = a.part[(int64_t)st.row * a.parts + i];
            lefts[i] = p.m == -INFINITY ? 0.0 : p.s * weight(p.m, st.p.m, a.c) * st.p.by;
        }
        __syncthreads();
        total = 0.0;
        for (int i = 0; i < a.parts; ++i) total += lefts[i];
    }
    const double want = (double)a.uniforms[first + n - 1] * total;
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
    if (tid == 0) chosen = -1;
    int tail = -1;                               // the last token of this lane's that has any weight
    for (int base = from; base < to; base += kPiece) {
        double r[8], local = 0.0;
        const int i0 = base + tid * 8;
        left8<DT>(a, st, residual, i0, to, r);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            local += r[k];
            if (r[k] > 0.0) tail = i0 + k;
        }
        double upto = local;
#pragma unroll
        for (int off = 1; off < kWave; off <<= 1) {
            const double v = __shfl_up(upto, off, kWave);
            if (lane >= off) upto += v;
        }
        __syncthreads();
        if (lane == kWave - 1) sums[wave] = upto;
        __syncthreads();
        double behind = before;
        for (int w = 0; w < wave; ++w) behind += sums[w];
        const double all = before + ((sums[0] + sums[1]) + (sums[2] + sums[3]));
        double c = behind + (upto - local);
        int hit = INT32_MAX;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            c += r[k];
            if (hit == INT32_MAX && c > want && r[k] > 0.0) hit = i0 + k;
        }
#pragma unroll
        for (int off = kWave / 2; off > 0; off >>= 1) hit = min(hit, __shfl_xor(hit, off, kWave));
        if (lane == 0) agreed[wave] = hit;
        __syncthreads();
        hit = min(min(agreed[0], agreed[1]), min(agreed[2], agreed[3]));
        if (hit != INT32_MAX) {
            if (tid == 0) chosen = hit;
            break;
        }
        before = all;
    }
    __syncthreads();
    if (chosen < 0) {                            // (uniform)
#pragma unroll
        for (int off = kWave / 2; off > 0; off >>= 1) tail = max(tail, __shfl_xor(tail, off, kWave));
        if (lane == 0) agreed[wave] = tail;
        __syncthreads();
        if (tid == 0) chosen = max(max(agreed[0], agreed[1]), max(agreed[2], agreed[3]));
    }
    if (tid == 0) {
        a.accepted[s] = at;
        a.out[st.row] = chosen;
        const float x = element<DT>(row_at<DT>(a.logits, st.row, a.stride), max(chosen, 0));
        a.logprobs[st.row] = (float)(((double)x - (double)st.p.m) * a.c * 0.69314718055994530942 + log(st.p.by));
    }
}

// Parts of a row: so that a call has about four blocks a compute unit, of 2048 columns at least and 8192 where there are enough.
int parts_of(int64_t rows, int64_t vocab, int &span) {
    const int64_t blocks = 4 * (int64_t)device_cu_count();
    span = rows * ((vocab + 4 * kPiece - 1) / (4 * kPiece)) >= blocks ? 4 * kPiece : kPiece;
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
    return rows * 2 * parts * 4 + seqs * parts * 2 + seqs;
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
    a.left = reinterpret_cast<double *>(a.part + 2 * rows * a.parts);
    a.arrived = reinterpret_cast<uint32_t *>(a.left + seqs * a.parts);
    hipStream_t stream = reinterpret_cast<hipStream_t>(stream_);
#define ODL_VERIFY(KERNEL, GRID)                                                                                              \
    do {                                                                                                                      \
        if (dtype == ODL_BF16 && greedy) hipLaunchKernelGGL((KERNEL<ODL_BF16, true>), GRID, dim3(kThreads), 0, stream, a);    \
        else if (dtype == ODL_BF16) hipLaunchKernelGGL((KERNEL<ODL_BF16, false>), GRID, dim3(kThreads), 0, stream, a);        \
        else if (greedy) hipLaunchKernelGGL((KERNEL<ODL_F32, true>), GRID, dim3(kThreads), 0, stream, a);                     \
        else hipLaunchKernelGGL((KERNEL<ODL_F32, false>), GRID, dim3(kThreads), 0, stream, a);                                \
    } while (0)
    if (rows > 0) ODL_VERIFY(draft_sums_kernel, dim3((unsigned)a.parts, (unsigned)rows, a.drafts ? 2u : 1u));
    if (seqs > 0) ODL_VERIFY(draft_verify_kernel, dim3(greedy ? 1u : (unsigned)a.parts, (unsigned)seqs));
#undef ODL_VERIFY
    return check_launch(who);
}
