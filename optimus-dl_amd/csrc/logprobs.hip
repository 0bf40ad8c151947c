// Log probabilities of given tokens from the logits of a head, with the entropy of each row and its top alternatives, and the
// gradient of the logits.  With d_j = (l_j - m) / T, m the row's maximum, s = sum e^d_j, q = sum e^d_j d_j:
//   logprob = d_t - ln s,  entropy = ln s - q / s (both terms >= 0: nothing cancels),  top_i = d_i - ln s
//   p_j = e^d_j / s,  dl_j = [A (j == t) + sum_i C_i (j == id_i) - p_j (A + sum_i C_i) - B p_j (ln p_j + entropy)] / T
// for gradients A of the logprob, B of the entropy, C_i of the top alternatives.
//
// The forward reads a row once, with a running maximum and the two sums of it per lane.  The top k cost no work in that pass:
// the k-th largest of the lanes' maxima is a lower bound of the k-th largest logit, and only lanes whose maximum reaches it can hold
// one; their share of the row (k lanes of 256, mostly) is read again and what reaches the bound is ranked.
// Rows are read and written with 16-byte accesses at any alignment (rows of an odd number of columns begin anywhere).
// Bound by HBM for large calls (8 to 12 operations an element, one of them an exponential), by latency for a few rows.
#include "common.h"

#pragma clang fp contract(off)

namespace odl {
namespace {

constexpr int kParts = ODL_FP8_AMAX_PARTS;
constexpr int kThreads = 256;
constexpr int kMaxTop = ODL_FP8_LOGPROBS_MAX_TOP;
constexpr int kMaxSplits = ODL_FP8_LOGPROBS_MAX_SPLITS;
constexpr int kCand = 1024;                      // candidates of a section that are ranked at once
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kFar = 1e30f;                    // exponents are cut off here: finite times e^-far is 0, infinity times 0 is not

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

// Running maximum m (never below -FLT_MAX, so that differences stay finite), s = sum 2^d, q = sum 2^d d, d = (l - m) * c,
// c = log2(e) / T.
struct Softmax {
    float m = -FLT_MAX, s = 0.0f, q = 0.0f;
    __device__ __forceinline__ void move_to(float to, float c) {
        const float delta = fminf((to - m) * c, kFar), f = __builtin_amdgcn_exp2f(-delta);
        q = f * __fmaf_rn(-delta, s, q);
        s *= f;
        m = to;
    }
    __device__ __forceinline__ void add(const Softmax &o, float c) {
        Softmax b = o;
        const float to = fmaxf(m, b.m);
        move_to(to, c);
        b.move_to(to, c);
        s += b.s;
        q += b.q;
    }
    __device__ __forceinline__ void take(float l, float c) {       // l <= m
        const float d = (l - m) * c, e = __builtin_amdgcn_exp2f(d);
        s += e;
        q = __fmaf_rn(e, fmaxf(d, -kFar), q);
    }
};

__device__ __forceinline__ Softmax wave_softmax(Softmax a, float c) {
#pragma unroll
    for (int off = kWave / 2; off > 0; off >>= 1) {
        Softmax b;
        b.m = __shfl_xor(a.m, off, kWave);
        b.s = __shfl_xor(a.s, off, kWave);
        b.q = __shfl_xor(a.q, off, kWave);
        a.add(b, c);
    }
    return a;
}

struct Row {                                     // what a row answers
    float m, log_s, entropy;
};

// (a sum of 0: every logit is -inf)
__device__ __forceinline__ Row answer(const Softmax &a) {
    Row r;
    r.m = a.m;
    r.log_s = a.s == 0.0f ? -INFINITY : logf(a.s);
    r.entropy = a.s == 0.0f ? 0.0f : r.log_s - a.q * kLn2 / a.s;
    return r;
}

__device__ __forceinline__ float log_prob(float l, const Row &r, float inv_t) {
    if (r.log_s == -INFINITY) return -INFINITY;
    return (l - r.m) * inv_t - r.log_s;
}

__device__ __forceinline__ bool before(float v, int i, float w, int j) { return v > w || (v == w && i < j); }

struct Forward {
    const void *logits;
    const int64_t *targets;
    int64_t rows, stride, ignore_index;
    int vocab, top_k, splits, section;           // a section: columns of a block, a multiple of 8
    float inv_t;
    float *logprobs, *entropy, *stats, *top_logprobs;
    int64_t *top_ids;
    float *part_sums, *part_values;              // splits > 1: [rows][splits][3], [rows][splits][top_k]
    int *part_ids;
};

__device__ __forceinline__ void write_ignored(const Forward &a, int64_t row) {
    if (threadIdx.x == 0) {
        a.logprobs[row] = 0.0f;
        a.entropy[row] = 0.0f;
        if (a.stats) { a.stats[row] = 0.0f; a.stats[a.rows + row] = 0.0f; }
    }
    for (int i = threadIdx.x; i < a.top_k; i += kThreads) {
        a.top_logprobs[row * a.top_k + i] = 0.0f;
        a.top_ids[row * a.top_k + i] = -1;
    }
}

template <int DT>
__device__ __forceinline__ void write_row(const Forward &a, int64_t row, int64_t target, const Row &r) {
    float lp = __builtin_nanf("");
    if (target >= 0 && target < a.vocab)
        lp = log_prob(one<DT>(reinterpret_cast<const typename Elem<DT>::T *>(a.logits) + row * a.stride + target), r, a.inv_t);
    a.logprobs[row] = lp;
    a.entropy[row] = r.entropy;
    if (a.stats) { a.stats[row] = r.m; a.stats[a.rows + row] = r.log_s; }
}

__device__ __forceinline__ void write_top(const Forward &a, int64_t row, int rank, float v, int id, const Row &r) {
    const bool sound = r.log_s == r.log_s;       // a row with NaN or +inf has no order
    a.top_logprobs[row * a.top_k + rank] = sound ? log_prob(v, r, a.inv_t) : __builtin_nanf("");
    a.top_ids[row * a.top_k + rank] = sound ? id : -1;
}

// One block for each row and section of its columns.
template <int DT>
__global__ __launch_bounds__(kThreads) void token_logprobs_kernel(const Forward a) {
    typedef typename Elem<DT>::T T;
    constexpr int U = 4;
    __shared__ float sums[kThreads / kWave][3], cand_v[kCand], bound;
    __shared__ __attribute__((aligned(16))) float lane_top[kThreads];
    __shared__ int cand_i[kCand], lanes[kThreads], n_lanes, n_cand;
    const int tid = threadIdx.x;
    const int64_t row = blockIdx.x / a.splits;
    const int sec = (int)(blockIdx.x - row * a.splits);
    const int64_t target = a.targets[row];
    if (target == a.ignore_index) {              // (not read)
        if (a.splits == 1) write_ignored(a, row);
        return;
    }
    const int first = sec * a.section, cols = min(a.section, a.vocab - first);
    const T *p = reinterpret_cast<const T *>(a.logits) + row * a.stride + first;
    const int n = cols / 8, tail = cols % 8;
    const float c = a.inv_t * kLog2e;
    Softmax run;
    float top = -INFINITY;
    for (int i = tid; i < n; i += U * kThreads) {
        Chunk<DT> in[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (i + u * kThreads < n) in[u].load(p + (int64_t)(i + u * kThreads) * 8);
            else in[u].fill();
        }
        float f[U][8], most = -INFINITY;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            in[u].widen(f[u]);
#pragma unroll
            for (int e = 0; e < 8; ++e) most = fmaxf(most, f[u][e]);
        }
        top = fmaxf(top, most);
        run.move_to(fmaxf(run.m, most), c);
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int e = 0; e < 8; ++e) run.take(f[u][e], c);
    }
    if (tid < tail) {
        const float l = one<DT>(p + n * 8 + tid);
        top = fmaxf(top, l);
        run.move_to(fmaxf(run.m, l), c);
        run.take(l, c);
    }
    run = wave_softmax(run, c);
    if (tid % kWave == 0) {
        sums[tid / kWave][0] = run.m;
        sums[tid / kWave][1] = run.s;
        sums[tid / kWave][2] = run.q;
    }
    if (a.top_k) {
        lane_top[tid] = top;
        if (tid == 0) n_lanes = n_cand = 0;
    }
    __syncthreads();
    run = Softmax{sums[0][0], sums[0][1], sums[0][2]};
#pragma unroll
    for (int w = 1; w < kThreads / kWave; ++w) run.add(Softmax{sums[w][0], sums[w][1], sums[w][2]}, c);
    const Row r = answer(run);
    if (tid == 0) {
        if (a.splits == 1) {
            write_row<DT>(a, row, target, r);
        } else {
            float *o = a.part_sums + blockIdx.x * (int64_t)3;
            o[0] = run.m; o[1] = run.s; o[2] = run.q;
        }
    }
    if (!a.top_k) return;

    auto put = [&](int rank, float v, int id) {
        if (a.splits == 1) {
            write_top(a, row, rank, v, id, r);
        } else {
            a.part_values[blockIdx.x * (int64_t)a.top_k + rank] = v;
            a.part_ids[blockIdx.x * (int64_t)a.top_k + rank] = id;
        }
    };
    {                                            // the k-th largest of the lanes' maxima
        int rank = 0;
        for (int j = 0; j < kThreads; j += 4) {
            const float4 o = *reinterpret_cast<const float4 *>(lane_top + j);
            rank += before(o.x, j, top, tid) + before(o.y, j + 1, top, tid) + before(o.z, j + 2, top, tid) + before(o.w, j + 3, top, tid);
        }
        if (rank == a.top_k - 1) bound = top;
    }
    __syncthreads();
    const float least = bound;
    if (top >= least) lanes[atomicAdd(&n_lanes, 1)] = tid;
    __syncthreads();
    auto offer = [&](float v, int col) {
        if (v >= least) {
            const int at = atomicAdd(&n_cand, 1);
            if (at < kCand) { cand_v[at] = v; cand_i[at] = first + col; }
        }
    };
    const int per = (n + kThreads - 1) / kThreads, total = n_lanes * per;
    for (int i = tid; i < total; i += kThreads) {
        const int chunk = lanes[i / per] + (i % per) * kThreads;
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
        for (int i = tid; i < found; i += kThreads) {
            const float v = cand_v[i];
            const int id = cand_i[i];
            int rank = 0;
            for (int j = 0; j < found; ++j) rank += before(cand_v[j], cand_i[j], v, id);
            if (rank < a.top_k) put(rank, v, id);
        }
        // (fewer than k: a section of fewer columns, or NaN in the row)
        for (int i = found + tid; i < a.top_k; i += kThreads) put(i, -INFINITY, INT_MAX);
        return;
    }
    // More than a thousand logits share the bound (rows that are masked almost everywhere, say): the largest behind the last one
    // found, k times over.
    float last_v = INFINITY;
    int last_i = -1;
    for (int k = 0; k < a.top_k; ++k) {
        float best_v = -INFINITY;
        int best_i = INT_MAX;
        auto look = [&](float v, int id) {
            if (before(last_v, last_i, v, id) && before(v, id, best_v, best_i)) { best_v = v; best_i = id; }
        };
        for (int i = tid; i < n; i += kThreads) {
            Chunk<DT> in;
            in.load(p + (int64_t)i * 8);
            float f[8];
            in.widen(f);
#pragma unroll
            for (int e = 0; e < 8; ++e) look(f[e], first + i * 8 + e);
        }
        if (tid < tail) look(one<DT>(p + n * 8 + tid), first + n * 8 + tid);
#pragma unroll
        for (int off = kWave / 2; off > 0; off >>= 1) {
            const float v = __shfl_xor(best_v, off, kWave);
            const int id = __shfl_xor(best_i, off, kWave);
            if (before(v, id, best_v, best_i)) { best_v = v; best_i = id; }
        }
        __syncthreads();                         // (cand_v and cand_i are read by everybody in the round before)
        if (tid % kWave == 0) { cand_v[tid / kWave] = best_v; cand_i[tid / kWave] = best_i; }
        __syncthreads();
        best_v = cand_v[0];
        best_i = cand_i[0];
        for (int w = 1; w < kThreads / kWave; ++w)
            if (before(cand_v[w], cand_i[w], best_v, best_i)) { best_v = cand_v[w]; best_i = cand_i[w]; }
        last_v = best_v;
        last_i = best_i;
        if (tid == 0) put(k, best_v, best_i);
    }
}

// Rows whose columns were split: one block joins the sections of a row, in their order.
template <int DT>
__global__ __launch_bounds__(kThreads) void token_logprobs_join_kernel(const Forward a) {
    __shared__ float cand_v[kMaxSplits * kMaxTop], least;
    __shared__ int cand_i[kMaxSplits * kMaxTop], n_cand;
    const int tid = threadIdx.x;
    const int64_t row = blockIdx.x, target = a.targets[row];
    if (target == a.ignore_index) {
        write_ignored(a, row);
        return;
    }
    const float c = a.inv_t * kLog2e;
    Softmax run;
    if (tid % kWave < a.splits) {                // a lane for each section, at most a wave of them; every wave does the same
        const float *o = a.part_sums + (row * a.splits + tid % kWave) * 3;
        run.m = o[0]; run.s = o[1]; run.q = o[2];
    }
    run = wave_softmax(run, c);
    const Row r = answer(run);
    if (tid == 0) write_row<DT>(a, row, target, r);
    if (!a.top_k) return;
    const float *values = a.part_values + row * a.splits * a.top_k;
    const int *ids = a.part_ids + row * a.splits * a.top_k;
    if (tid < kWave) {                           // the k-th largest of any section is a lower bound
        float v = tid < a.splits ? values[tid * a.top_k + a.top_k - 1] : -INFINITY;
#pragma unroll
        for (int off = kWave / 2; off > 0; off >>= 1) v = fmaxf(v, __shfl_xor(v, off, kWave));
        if (tid == 0) { least = v; n_cand = 0; }
    }
    __syncthreads();
    for (int i = tid; i < a.splits * a.top_k; i += kThreads)
        if (values[i] >= least && ids[i] != INT_MAX) {
            const int at = atomicAdd(&n_cand, 1);
            cand_v[at] = values[i];
            cand_i[at] = ids[i];
        }
    __syncthreads();
    const int found = n_cand;
    for (int i = tid; i < found; i += kThreads) {
        const float v = cand_v[i];
        const int id = cand_i[i];
        int rank = 0;
        for (int j = 0; j < found; ++j) rank += before(cand_v[j], cand_i[j], v, id);
        if (rank < a.top_k) write_top(a, row, rank, v, id, r);
    }
    for (int i = found + tid; i < a.top_k; i += kThreads) write_top(a, row, i, -INFINITY, -1, r);
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

constexpr int kBwdThreads = 512, kMarks = 128;

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
        const float m = a.stats[row], log_s = a.stats[a.rows + row];
        const bool nothing = target == a.ignore_index || log_s == -INFINITY;
        float sum = a.d_logprobs ? a.d_logprobs[row] : 0.0f;
        const float given = sum * a.inv_t, b = a.d_entropy ? a.d_entropy[row] : 0.0f;
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
            for (int i = 0; i < a.top_k; ++i) sum += top_d[i];
        }
        float k0 = -a.inv_t * __fmaf_rn(b, a.entropy[row] - log_s, sum);
        const float k1 = -a.inv_t * b * a.inv_t, c = a.inv_t * kLog2e, l2 = log_s * kLog2e;
        if (target < 0 || target >= a.vocab) k0 = __builtin_nanf("");          // no such token: its log probability is NaN too
        const int t_chunk = target >= 0 && target < a.vocab ? (int)target / 8 : -1;
        auto gradient = [&](float l) {
            const float d = l - m, p = __builtin_amdgcn_exp2f(__fmaf_rn(d, c, -l2));
            return p * __fmaf_rn(fmaxf(d, -kFar), k1, k0);
        };
        // gradients of a chunk in which the target or a top alternative may lie, or that ends behind the vocabulary
        auto special = [&](int chunk, float (&f)[8]) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int col = chunk * 8 + e;
                if (chunk == t_chunk && col == (int)target) f[e] += given;
                if constexpr (TOP)
                    for (int i = 0; i < a.top_k; ++i)
                        if (top_i[i] == col) f[e] = __fmaf_rn(top_d[i], a.inv_t, f[e]);
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
                        if (top_i[i] == col) f = __fmaf_rn(top_d[i], a.inv_t, f);
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
    am = block_max_u32(DT == ODL_BF16 ? fold_u16x2_to_f32bits(am) : am, red);
    if (tid == 0) a.parts[blockIdx.x] = bits_to_float(am);
    if (blockIdx.x == 0)
        for (int j = (int)gridDim.x + tid; j < kParts; j += kBwdThreads) a.parts[j] = 0.0f;
}

int check(const char *who, int dtype, int64_t rows, int64_t stride, int64_t padded, int64_t vocab, int top_k, float inv_t) {
    if (rows < 0 || stride < 0) return set_error(ODL_ERR_ARG, "%s: negative shape", who);
    if (dtype != ODL_BF16 && dtype != ODL_F32) return set_error(ODL_ERR_ARG, "%s: dtype %d", who, dtype);
    if (vocab < 1 || vocab > padded || padded > (1 << 24)) return set_error(ODL_ERR_SHAPE, "%s: %lld of %lld columns (1 to 2^24)", who, (long long)vocab, (long long)padded);
    if (rows >= (1 << 24)) return set_error(ODL_ERR_SHAPE, "%s: %lld rows (up to 2^24 - 1)", who, (long long)rows);
    if (top_k < 0 || top_k > kMaxTop || top_k > vocab) return set_error(ODL_ERR_ARG, "%s: top_k %d (0 to %d, and to the vocabulary)", who, top_k, kMaxTop);
    if (!(inv_t > 0.0f) || __builtin_isinf(inv_t)) return set_error(ODL_ERR_ARG, "%s: the temperature must be positive and finite", who);
    return ODL_OK;
}

}  // namespace
}  // namespace odl

using namespace odl;

// Sections of a row: enough blocks for four on every compute unit, none of fewer than 2048 columns (a chunk for every lane).
extern "C" int odl_fp8_token_logprobs_splits(int64_t rows, int64_t vocab) {
    if (rows < 1 || vocab < 1) return 1;
    const int64_t want = (4 * (int64_t)device_cu_count() + rows - 1) / rows, most = (vocab + 2047) / 2048;
    int64_t s = want < most ? want : most;
    s = s < kMaxSplits ? s : kMaxSplits;
    return (int)(s < 1 ? 1 : s);
}

extern "C" int odl_fp8_token_logprobs(const void *logits, int dtype, int64_t rows, int64_t stride, int64_t vocab, const int64_t *targets,
                                      int64_t ignore_index, float inv_temperature, int top_k, float *logprobs, float *entropy, float *stats,
                                      float *top_logprobs, int64_t *top_ids, int splits, float *workspace, odl_stream_t stream_) {
    hipStream_t stream = reinterpret_cast<hipStream_t>(stream_);
    if (const int rc = check("odl_fp8_token_logprobs", dtype, rows, stride, vocab, vocab, top_k, inv_temperature)) return rc;
    if (rows == 0) return ODL_OK;
    if (!logits || !targets || !logprobs || !entropy || (top_k && (!top_logprobs || !top_ids)))
        return set_error(ODL_ERR_ARG, "odl_fp8_token_logprobs: null pointer");
    if (splits < 1 || splits > kMaxSplits || (splits > 1 && !workspace))
        return set_error(ODL_ERR_ARG, "odl_fp8_token_logprobs: %d sections (1 to %d; more than one need a workspace)", splits, kMaxSplits);
    if (rows * splits >= (1 << 24))              // (lanes of a launch are counted in 32 bits)
        return set_error(ODL_ERR_SHAPE, "odl_fp8_token_logprobs: %lld rows of %d sections (up to 2^24 - 1 blocks)", (long long)rows, splits);
    const int64_t chunks = (vocab + 7) / 8, section = (chunks + splits - 1) / splits * 8;
    splits = (int)((vocab + section - 1) / section);              // (no section is empty)
    Forward a = {};
    a.logits = logits; a.targets = targets; a.rows = rows; a.stride = stride; a.ignore_index = ignore_index;
    a.vocab = (int)vocab; a.top_k = top_k; a.splits = splits; a.section = (int)section; a.inv_t = inv_temperature;
    a.logprobs = logprobs; a.entropy = entropy; a.stats = stats; a.top_logprobs = top_logprobs; a.top_ids = top_ids;
    a.part_sums = workspace;
    if (splits > 1 && top_k) {
        a.part_values = workspace + rows * splits * 3;
        a.part_ids = reinterpret_cast<int *>(a.part_values + rows * splits * top_k);
    }
    const dim3 grid((unsigned)(rows * splits));
    if (dtype == ODL_BF16) hipLaunchKernelGGL(token_logprobs_kernel<ODL_BF16>, grid, dim3(kThreads), 0, stream, a);
    else hipLaunchKernelGGL(token_logprobs_kernel<ODL_F32>, grid, dim3(kThreads), 0, stream, a);
    if (splits > 1) {
        if (dtype == ODL_BF16) hipLaunchKernelGGL(token_logprobs_join_kernel<ODL_BF16>, dim3((unsigned)rows), dim3(kThreads), 0, stream, a);
        else hipLaunchKernelGGL(token_logprobs_join_kernel<ODL_F32>, dim3((unsigned)rows), dim3(kThreads), 0, stream, a);
    }
    return check_launch("odl_fp8_token_logprobs");
}

extern "C" int odl_fp8_token_logprobs_bwd(const void *logits, int dtype, int64_t rows, int64_t stride, int64_t vocab, int64_t padded,
                                          const int64_t *targets, int64_t ignore_index, float inv_temperature, int top_k, const int64_t *top_ids,
                                          const float *stats, const float *entropy, const float *d_logprobs, const float *d_entropy,
                                          const float *d_top, void *dlogits, float *parts, odl_stream_t stream_) {
    hipStream_t stream = reinterpret_cast<hipStream_t>(stream_);
    if (const int rc = check("odl_fp8_token_logprobs_bwd", dtype, rows, stride, padded, vocab, top_k, inv_temperature)) return rc;
    if (!parts || (rows > 0 && (!logits || !targets || !stats || !entropy || !dlogits)) || (d_top && top_k && !top_ids))
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
