// New queries, keys and values of a step on their way into a paged cache:
//   n = x * r * w, r = 1 / sqrt(mean(x^2) + eps)  (where a norm's weight is given),  (a, b) -> (a cos - b sin, a sin + b cos),  one rounding
// A row of a head is held by 16 lanes, 8 elements each; pairs of a rotation lie in one lane (interleaved) or come from another lane of the row
// (halves).  Everything but the mean of squares is a fixed order of fp32 operations, and that is held in 64 bits: the result does not
// depend on how the sum is cut, so that codes of 8 bits are the same wherever they are computed this way.
//
// HBM bounds it: 4 bytes an element of queries, 4 (bf16) or 3 (codes) of keys and values.  Everything a row needs is in its lanes, so that a token's rows go over as
// many blocks as they fill, and one token's latency is that of one chain of loads: offsets, length, page.  Measured (calls in a row): 1 token 7.6 us and 256 tokens 7.5 (the
// host's; the kernel 3.0 and 4.8), 7331 tokens of 32 + 2 x 8 heads of 128 42.6 us, 4.3 TB/s (a large copy: 5.1).
#include "paged.h"

#pragma clang fp contract(off)

namespace odl {
namespace {

bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
bool power_of_two(int64_t v) { return v > 0 && (v & (v - 1)) == 0; }

}  // namespace

int take_paged(const char *who, const odl_fp8_paged_cache *c, const odl_fp8_paged_batch *b, Paged &to) {
    if (!c || !b) return set_error(ODL_ERR_ARG, "%s: null pointer", who);
    if (c->pages < 0 || c->kv_heads < 1 || b->seqs < 0 || b->rows < 0 || b->width < 0) return set_error(ODL_ERR_ARG, "%s: negative or empty shape", who);
    if ((c->pages > 0 && (!c->keys || !c->values)) || (c->e4m3 && (!c->key_scale || !c->value_scale)))
        return set_error(ODL_ERR_ARG, "%s: a null pointer for the cache", who);
    if (!b->offsets || (b->seqs > 0 && (!b->lengths || (b->width > 0 && !b->table)))) return set_error(ODL_ERR_ARG, "%s: a null pointer for the batch", who);
    if (c->head_dim < 16 || c->head_dim > 128 || c->head_dim % 16) return set_error(ODL_ERR_SHAPE, "%s: heads of %lld (16 to 128, a multiple of 16)", who, (long long)c->head_dim);
    if (!power_of_two(c->page_size) || c->page_size > 1 << 20) return set_error(ODL_ERR_SHAPE, "%s: pages of %lld tokens (a power of two up to 2^20)", who, (long long)c->page_size);
    if (c->pages > INT32_MAX || c->kv_heads > 1024 || b->seqs > 1 << 20 || b->rows > 1 << 24) return set_error(ODL_ERR_SHAPE, "%s: more pages, heads, sequences or rows than a call takes", who);
    if (b->width > (1 << 30) / c->page_size) return set_error(ODL_ERR_SHAPE, "%s: a page table for more than 2^30 tokens", who);
    const int size = c->e4m3 ? 1 : 2;
    if (!aligned16(c->keys) || !aligned16(c->values)) return set_error(ODL_ERR_SHAPE, "%s: the cache must be 16-byte aligned", who);
    for (int i = 0; i < 3; ++i)
        if ((c->key_strides[i] * size) % 16 || (c->value_strides[i] * size) % 16 || c->key_strides[i] < 0 || c->value_strides[i] < 0)
            return set_error(ODL_ERR_SHAPE, "%s: strides of the cache must be multiples of 16 bytes", who);
    to.keys = static_cast<uint8_t *>(c->keys);
    to.values = static_cast<uint8_t *>(c->values);
    to.key_scale = c->e4m3 ? c->key_scale : nullptr;
    to.value_scale = c->e4m3 ? c->value_scale : nullptr;
    to.k_page = c->key_strides[0] * size, to.k_head = c->key_strides[1] * size, to.k_tok = c->key_strides[2] * size;
    to.v_page = c->value_strides[0] * size, to.v_head = c->value_strides[1] * size, to.v_tok = c->value_strides[2] * size;
    to.table = b->table, to.offsets = b->offsets, to.lengths = b->lengths, to.table_stride = b->table_stride;
    to.seqs = (int)b->seqs, to.rows = (int)b->rows, to.pages = (int)c->pages, to.kv_heads = (int)c->kv_heads, to.dim = (int)c->head_dim;
    to.shift = __builtin_ctzll((uint64_t)c->page_size), to.e4m3 = c->e4m3 != 0, to.reach = (int)(b->width * c->page_size);
    return ODL_OK;
}

int check_strides(const char *who, const char *name, const void *p, const int64_t *strides, int64_t rows) {
    if (rows > 0 && (!p || !strides)) return set_error(ODL_ERR_ARG, "%s: null pointer for %s", who, name);
    if (rows > 0 && (!aligned16(p) || strides[0] % 8 || strides[1] % 8 || strides[0] < 0 || strides[1] < 0))
        return set_error(ODL_ERR_SHAPE, "%s: %s must be 16-byte aligned, with strides in multiples of 8", who, name);
    return ODL_OK;
}

namespace {

constexpr int kLanes = 16;                       // lanes of a row of a head
constexpr int kRows = 16;                        // rows that a block of 256 lanes holds at a time

struct Append {
    Paged p;
    const uint16_t *q, *k, *v;
    int64_t q_row, q_head, k_row, k_head, v_row, v_head;       // strides in elements
    const float *cos, *sin;
    const void *q_weight, *k_weight;
    double eps;
    int heads, half, interleaved, weight_bf16;
    uint16_t *out;
};

// A block has one token and 16 of its rows (queries, keys, values in this order).
__global__ __launch_bounds__(256) void append_kv_kernel(Append a) {
    const int t = blockIdx.x, slot = blockIdx.y * kRows + threadIdx.x / kLanes, c = threadIdx.x % kLanes, lane = threadIdx.x % kWave;
    const Paged &p = a.p;
    const int kv = p.kv_heads, count = a.heads + 2 * kv;
    const bool live = slot < count && c * 8 < p.dim;
    const bool is_q = slot < a.heads, is_v = slot >= a.heads + kv;
    const int head = is_q ? slot : is_v ? slot - a.heads - kv : slot - a.heads;
    const uint16_t *src = is_q ? a.q + t * a.q_row + head * a.q_head : is_v ? a.v + t * a.v_row + head * a.v_head : a.k + t * a.k_row + head * a.k_head;
    u32x4 raw = {0, 0, 0, 0};
    if (live) raw = *reinterpret_cast<const u32x4 *>(src + c * 8);

    // the token's sequence: how many of them end at or in front of it
    int s = 0;
    for (int s0 = 0; s0 < p.seqs; s0 += kWave) s += __popcll(__ballot(s0 + lane < p.seqs && p.offsets[s0 + lane + 1] <= t));
    s = __builtin_amdgcn_readfirstlane(s);
    if (s >= p.seqs) {                           // nobody's
        if (live && is_q) *reinterpret_cast<u32x4 *>(a.out + ((int64_t)t * a.heads + head) * p.dim + c * 8) = u32x4{0, 0, 0, 0};
        return;
    }
    const Run run = run_of(p, s);
    const int pos = p.lengths[s] - run.n + (t - run.first);
    const bool placed = t >= run.first && pos >= 0 && pos < p.reach;
    int page = -1;
    if (placed) page = p.table[s * p.table_stride + (pos >> p.shift)];

    float x[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) { x[2 * i] = bf16_lo(raw[i]); x[2 * i + 1] = bf16_hi(raw[i]); }
    const void *weight = is_q ? a.q_weight : is_v ? nullptr : a.k_weight;
    if (a.q_weight || a.k_weight) {
        double sum = 0.0;
#pragma unroll
        for (int i = 0; i < 8; ++i) sum += (double)x[i] * (double)x[i];
#pragma unroll
        for (int off = kLanes / 2; off > 0; off >>= 1) sum += __shfl_xor(sum, off, kWave);
        if (weight && live) {
            const float r = (float)(1.0 / sqrt(sum / (double)p.dim + a.eps));
            float w[8];
            if (a.weight_bf16) {
                uint32_t two[4];
                __builtin_memcpy(two, static_cast<const uint16_t *>(weight) + c * 8, sizeof(two));
#pragma unroll
                for (int i = 0; i < 4; ++i) { w[2 * i] = bf16_lo(two[i]); w[2 * i + 1] = bf16_hi(two[i]); }
            } else {
                __builtin_memcpy(w, static_cast<const float *>(weight) + c * 8, sizeof(w));
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = x[i] * r * w[i];
        }
    }
    if (a.half) {
        if (a.interleaved) {
            if (placed && !is_v && c * 8 < 2 * a.half) {
                float cs[4], sn[4];
                __builtin_memcpy(cs, a.cos + (int64_t)pos * a.half + c * 4, sizeof(cs));
                __builtin_memcpy(sn, a.sin + (int64_t)pos * a.half + c * 4, sizeof(sn));
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float u = x[2 * i], v = x[2 * i + 1];
                    x[2 * i] = u * cs[i] - v * sn[i];
                    x[2 * i + 1] = u * sn[i] + v * cs[i];
                }
            }
        } else {
            const int hc = a.half / 8, first = c < hc ? c : c - hc;            // chunks of a half, and the chunk's place in it
            float other[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) other[i] = __shfl(x[i], c < hc ? lane + hc : lane - hc, kWave);
            if (placed && !is_v && c < 2 * hc) {
                float cs[8], sn[8];
                __builtin_memcpy(cs, a.cos + (int64_t)pos * a.half + first * 8, sizeof(cs));
                __builtin_memcpy(sn, a.sin + (int64_t)pos * a.half + first * 8, sizeof(sn));
#pragma unroll
                for (int i = 0; i < 8; ++i) x[i] = c < hc ? x[i] * cs[i] - other[i] * sn[i] : other[i] * sn[i] + x[i] * cs[i];
            }
        }
    }
    if (!live) return;
    u32x4 rounded;
#pragma unroll
    for (int i = 0; i < 4; ++i) rounded[i] = pack_bf16x2(x[2 * i], x[2 * i + 1]);
    if (is_q) {
        *reinterpret_cast<u32x4 *>(a.out + ((int64_t)t * a.heads + head) * p.dim + c * 8) = placed ? rounded : u32x4{0, 0, 0, 0};
        return;
    }
    if (page < 0 || page >= p.pages) return;
    const int at = pos & ((1 << p.shift) - 1);
    uint8_t *to = is_v ? p.values + page * p.v_page + head * p.v_head + at * p.v_tok : p.keys + page * p.k_page + head * p.k_head + at * p.k_tok;
    if (p.e4m3) {
        const float scale = (is_v ? p.value_scale : p.key_scale)[head];
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = scale != 0.0f ? __fdiv_rn(x[i], scale) : x[i] != x[i] ? x[i] : 0.0f;           // (every code stands for 0; 0 / 0 would be none)
        *reinterpret_cast<u32x2 *>(to + c * 8) = u32x2{quantise4<ODL_FP8_E4M3>(x[0], x[1], x[2], x[3], 1.0f, 1.0f, 1.0f, 1.0f),
                                                        quantise4<ODL_FP8_E4M3>(x[4], x[5], x[6], x[7], 1.0f, 1.0f, 1.0f, 1.0f)};
    } else {
        *reinterpret_cast<u32x4 *>(to + c * 16) = rounded;
    }
}

}  // namespace
}  // namespace odl

using namespace odl;

extern "C" int odl_fp8_append_kv_typed(const void *q, const int64_t *q_strides, const void *k, const int64_t *k_strides, const void *v,
                                       const int64_t *v_strides, int64_t heads, const odl_fp8_paged_cache *cache, const odl_fp8_paged_batch *batch,
                                       const float *cos, const float *sin, int64_t positions, int64_t half, int interleaved, const void *q_weight,
                                       const void *k_weight, int weight_dtype, double eps, void *q_out, odl_stream_t stream_) {
    static const char who[] = "odl_fp8_append_kv";
    Append a;
    if (const int rc = take_paged(who, cache, batch, a.p)) return rc;
    if (heads < 1 || heads > 1024) return set_error(ODL_ERR_SHAPE, "%s: %lld heads (1 to 1024)", who, (long long)heads);
    if (half < 0 || 2 * half > a.p.dim || half % (interleaved ? 4 : 8)) return set_error(ODL_ERR_SHAPE, "%s: a rotation of %lld pairs in heads of %d (half a head at most, a multiple of %d)", who, (long long)half, a.p.dim, interleaved ? 4 : 8);
    if (half > 0 && (!cos || !sin)) return set_error(ODL_ERR_ARG, "%s: null pointer for the angles", who);
    if (half > 0 && positions < a.p.reach) return set_error(ODL_ERR_SHAPE, "%s: angles of %lld positions for a page table of %d", who, (long long)positions, a.p.reach);
    if (weight_dtype != ODL_F32 && weight_dtype != ODL_BF16) return set_error(ODL_ERR_ARG, "%s: weights of dtype %d", who, weight_dtype);
    const int64_t rows = batch->rows;
    if (const int rc = check_strides(who, "q", q, q_strides, rows)) return rc;
    if (const int rc = check_strides(who, "k", k, k_strides, rows)) return rc;
    if (const int rc = check_strides(who, "v", v, v_strides, rows)) return rc;
    if (rows == 0) return ODL_OK;
    if (rows * 256 > UINT32_MAX) return set_error(ODL_ERR_SHAPE, "%s: more rows than a launch has blocks (below 2^24)", who);
    if (!q_out || !aligned16(q_out)) return set_error(ODL_ERR_ARG, "%s: q_out must be a 16-byte aligned address", who);
    a.q = static_cast<const uint16_t *>(q), a.k = static_cast<const uint16_t *>(k), a.v = static_cast<const uint16_t *>(v);
    a.q_row = q_strides[0], a.q_head = q_strides[1], a.k_row = k_strides[0], a.k_head = k_strides[1], a.v_row = v_strides[0], a.v_head = v_strides[1];
    a.cos = cos, a.sin = sin, a.q_weight = q_weight, a.k_weight = k_weight, a.weight_bf16 = weight_dtype == ODL_BF16, a.eps = eps;
    a.heads = (int)heads, a.half = (int)half, a.interleaved = interleaved != 0, a.out = static_cast<uint16_t *>(q_out);
    const int64_t count = heads + 2 * a.p.kv_heads;
    hipLaunchKernelGGL(append_kv_kernel, dim3((unsigned)rows, (unsigned)((count + kRows - 1) / kRows)), dim3(256), 0, reinterpret_cast<hipStream_t>(stream_), a);
    return check_launch(who);
}

extern "C" int odl_fp8_append_kv(const void *q, const int64_t *q_strides, const void *k, const int64_t *k_strides, const void *v,
                                 const int64_t *v_strides, int64_t heads, const odl_fp8_paged_cache *cache, const odl_fp8_paged_batch *batch,
                                 const float *cos, const float *sin, int64_t positions, int64_t half, int interleaved, const float *q_weight,
                                 const float *k_weight, double eps, void *q_out, odl_stream_t stream) {
    return odl_fp8_append_kv_typed(q, q_strides, k, k_strides, v, v_strides, heads, cache, batch, cos, sin, positions, half, interleaved, q_weight,
                                   k_weight, ODL_F32, eps, q_out, stream);
}
