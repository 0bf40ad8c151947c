// The step of the residual stream between two blocks of a decoder, and its backward:
//   hh = h * rh, rh = 1 / sqrt(mean(h^2) + post_eps)      the norm behind the block (hh = h, rh = 1 without one)
//   y  = a * x + b * hh,  b = gate * post_weight          the gated block output on the scaled stream
//   z  = y * ry * weight, ry = 1 / sqrt(mean(y^2) + eps)  the norm in front of the next block
// z is of the fp32 y; y itself is rounded once, to the type of the stream.  Written apart these are four kernels and, with an
// fp32 stream and a bf16 block output, 34 bytes an element; here x and h are read once, y and z written once: 12 bytes.
//
// Backward, for gradients dy and dz.  y is computed again from x and h (which are read for the gradients anyway), so that
// nothing but rh and ry is kept and no rounding of y enters:
//   yh = y * ry, t = dz * weight, c2 = mean(t * yh)
//   e  = dy + ry * (t - yh * c2)                          the whole gradient of y
//   dx = a * e,  q = b * e,  c3 = mean(q * hh),  dh = rh * (q - hh * c3)     (dh = q without the norm behind the block)
//   d_weight = sum_rows dz * yh,  D = sum_rows e * hh,  d_post_weight = gate * D,  d_gate = post_weight * D
// c3 needs e and e needs c2; with k = b * hh it is ((S1 - ry * c2 * S2) / cols, S1 = sum k * (dy + ry * t), S2 = sum k * yh, so
// that one round of three row sums does for both means.
//
// Bound by HBM: 12 and 18 bytes an element (fp32 stream, bf16 block output) against some 10 and 40 operations.  16 to 512 lanes hold a row, two
// chunks of 8 elements a lane at most: the row is read once, the next one is on its way, and the weights of a lane's columns and the sums of
// their gradients stay in its registers from row to row.  8192 x 4096, fp32 / bf16: forward 76 us (5.3 TB/s; a copy reaches 5.1), backward
// 112 us (5.4 TB/s) and 5 us for the sums of its slabs; 4016 x 2048 in bf16 16, 23 and 4; one row of 4096 3.4, latency of its loads and sums.
// An fp32 block output beside an fp32 stream: 14 and 22 bytes an element, 8192 x 4096 forward and backward 234 us, 4096 x 8192 263 (5.2 and 4.6 TB/s; rows
// of more than 4096 spill 52 bytes a lane in the backward: 16 columns of six arrays).
#include "common.h"

#pragma clang fp contract(off)

namespace odl {
namespace {

constexpr int kParts = ODL_FP8_AMAX_PARTS;
constexpr int kSlabs = ODL_FP8_RESIDUAL_NORM_SLABS;

template <int T> constexpr int kVecs = T == ODL_BF16 ? 1 : 2;       // 16-byte vectors of 8 elements

template <int T>
__device__ __forceinline__ void load8(const void *base, int64_t chunk, bool ok, u32x4 (&raw)[kVecs<T>]) {
    const u32x4 *p = reinterpret_cast<const u32x4 *>(base) + chunk * kVecs<T>;
#pragma unroll
    for (int v = 0; v < kVecs<T>; ++v) raw[v] = ok ? __builtin_nontemporal_load(p + v) : u32x4{0, 0, 0, 0};
}

template <int T>
__device__ __forceinline__ void widen8(const u32x4 (&raw)[kVecs<T>], float (&f)[8]) {
    if constexpr (T == ODL_BF16) {
#pragma unroll
        for (int q = 0; q < 4; ++q) { f[2 * q] = bf16_lo(raw[0][q]); f[2 * q + 1] = bf16_hi(raw[0][q]); }
    } else {
#pragma unroll
        for (int q = 0; q < 8; ++q) f[q] = bits_to_float(raw[q / 4][q % 4]);
    }
}

template <int T>
__device__ __forceinline__ void store8(void *base, int64_t chunk, const float (&f)[8]) {
    u32x4 *p = reinterpret_cast<u32x4 *>(base) + chunk * kVecs<T>;
    if constexpr (T == ODL_BF16) {
        *p = u32x4{pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7])};
    } else {
#pragma unroll
        for (int v = 0; v < 2; ++v)
            p[v] = u32x4{float_to_bits(f[4 * v]), float_to_bits(f[4 * v + 1]), float_to_bits(f[4 * v + 2]), float_to_bits(f[4 * v + 3])};
    }
}

// Sums over the LPR lanes of a row, in every lane of it.  Up to a wave: xor butterfly.  Several waves: their sums through
// LDS in wave order; `turn` alternates between two buffers, so that a wave may still read one sum while another writes the
// next one's (a buffer is written again only behind the other one's barrier).
template <int LPR, int N>
__device__ __forceinline__ void row_sums(float (&v)[N], float *lds, int &turn) {
    constexpr int kLanes = LPR < kWave ? LPR : kWave;
#pragma unroll
    for (int off = kLanes / 2; off > 0; off >>= 1)
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] += __shfl_xor(v[i], off, kWave);
    if constexpr (LPR > kWave) {
        constexpr int kWaves = LPR / kWave;
        float *buf = lds + turn * N * kWaves;
        turn ^= 1;
        if (threadIdx.x % kWave == 0)
#pragma unroll
            for (int i = 0; i < N; ++i) buf[i * kWaves + threadIdx.x / kWave] = v[i];
        __syncthreads();
#pragma unroll
        for (int i = 0; i < N; ++i) {
            float s = buf[i * kWaves];
#pragma unroll
            for (int w = 1; w < kWaves; ++w) s += buf[i * kWaves + w];
            v[i] = s;
        }
    }
}

// How rows lie on a block: LPR lanes hold a row, lane l of them the chunks of 8 elements l, l + LPR, ..  (CPT of them), so a
// lane owns the same columns in every row and keeps their weights in registers.
template <int LPR>
struct Rows {
    static constexpr int kThreads = LPR > 256 ? LPR : 256;
    static constexpr int kPerBlock = kThreads / LPR;
};

// weights of a lane's columns: b without a scalar gate (that is `gs`), and the next norm's weight
template <int CPT, int LPR>
__device__ __forceinline__ void lane_weights(const float *weight, const float *post_weight, const float *gate, bool gate_scalar, int lane,
                                             int nchunk, float (&wv)[CPT][8], float (&wn)[CPT][8]) {
    auto take = [&](const float *from, float (&to)[CPT][8], float past) {
#pragma unroll
        for (int j = 0; j < CPT; ++j) {
            const int c = lane + j * LPR;
            if (c < nchunk) __builtin_memcpy(to[j], from + c * 8, sizeof(to[j]));
            else
#pragma unroll
                for (int e = 0; e < 8; ++e) to[j][e] = past;
        }
    };
    float g[CPT][8];
    take(weight, wn, 0.0f);
    const bool channels = gate && !gate_scalar;
    if (channels) take(gate, g, 0.0f);
    if (post_weight) {
        take(post_weight, wv, 0.0f);
    } else {
#pragma unroll
        for (int j = 0; j < CPT; ++j)
#pragma unroll
            for (int e = 0; e < 8; ++e) wv[j][e] = 1.0f;
    }
    if (channels) {
#pragma unroll
        for (int j = 0; j < CPT; ++j)
#pragma unroll
            for (int e = 0; e < 8; ++e) wv[j][e] *= g[j][e];
    }
}

template <int XT, int HT, int LPR, int CPT>
__global__ __launch_bounds__(Rows<LPR>::kThreads) void residual_norm_kernel(
    const void *__restrict__ x, const void *__restrict__ h, const float *__restrict__ weight, const float *__restrict__ post_weight,
    const float *__restrict__ gate, int gate_scalar, int64_t rows, int cols, float a, float eps, float post_eps, void *__restrict__ y,
    void *__restrict__ z, float *__restrict__ stats, float *__restrict__ parts) {
    constexpr int kThreads = Rows<LPR>::kThreads, RPB = Rows<LPR>::kPerBlock;
    __shared__ float lds[2 * (LPR / kWave + 1)];
    __shared__ uint32_t red[kThreads / kWave];
    const int lane = threadIdx.x % LPR, nchunk = cols / 8;
    const int64_t step = (int64_t)gridDim.x * RPB;
    const float gs = gate && gate_scalar ? gate[0] : 1.0f;
    u32x4 nx[CPT][kVecs<XT>], nh[CPT][kVecs<HT>];
    auto fetch = [&](int64_t row) {
#pragma unroll
        for (int j = 0; j < CPT; ++j) {
            const int c = lane + j * LPR;
            const bool ok = row < rows && c < nchunk;
            load8<XT>(x, row * nchunk + c, ok, nx[j]);
            load8<HT>(h, row * nchunk + c, ok, nh[j]);
        }
    };
    int turn = 0;
    uint32_t am = 0;
    int64_t row = (int64_t)blockIdx.x * RPB + threadIdx.x / LPR;
    fetch(row);
    float wv[CPT][8], wn[CPT][8];
    lane_weights<CPT, LPR>(weight, post_weight, gate, gate_scalar, lane, nchunk, wv, wn);
    for (int64_t row0 = (int64_t)blockIdx.x * RPB; row0 < rows; row0 += step, row += step) {      // the same trips for every lane
        float yf[CPT][8], hf[CPT][8];
#pragma unroll
        for (int j = 0; j < CPT; ++j) {
            widen8<XT>(nx[j], yf[j]);
            widen8<HT>(nh[j], hf[j]);
        }
        fetch(row + step);                                     // (rows past the end load nothing)
        float rh = 1.0f;
        if (post_weight) {
            float s[1] = {0.0f};
#pragma unroll
            for (int j = 0; j < CPT; ++j)
#pragma unroll
                for (int e = 0; e < 8; ++e) s[0] = __fmaf_rn(hf[j][e], hf[j][e], s[0]);
            row_sums<LPR, 1>(s, lds, turn);
            rh = 1.0f / __builtin_sqrtf(s[0] / (float)cols + post_eps);
        }
        float s[1] = {0.0f};
#pragma unroll
        for (int j = 0; j < CPT; ++j)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                yf[j][e] = __fmaf_rn(gs * wv[j][e], hf[j][e] * rh, a * yf[j][e]);
                s[0] = __fmaf_rn(yf[j][e], yf[j][e], s[0]);
            }
        row_sums<LPR, 1>(s, lds, turn);
        const float ry = 1.0f / __builtin_sqrtf(s[0] / (float)cols + eps);
        if (row < rows) {
            if (lane == 0 && stats) {
                stats[row] = rh;
                stats[rows + row] = ry;
            }
#pragma unroll
            for (int j = 0; j < CPT; ++j) {
                const int c = lane + j * LPR;
                if (c < nchunk) {
                    store8<XT>(y, row * nchunk + c, yf[j]);
                    uint32_t o[4];
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        o[q] = pack_bf16x2(yf[j][2 * q] * ry * wn[j][2 * q], yf[j][2 * q + 1] * ry * wn[j][2 * q + 1]);
                        am = max_u16x2(am, abs_bf16x2(o[q]));
                    }
                    reinterpret_cast<u32x4 *>(z)[row * nchunk + c] = u32x4{o[0], o[1], o[2], o[3]};
                }
            }
        }
    }
    if (!parts) return;
    am = block_max_u32(fold_u16x2_to_f32bits(am), red);
    if (threadIdx.x == 0) parts[blockIdx.x] = bits_to_float(am);
    if (blockIdx.x == 0)
        for (int j = (int)gridDim.x + threadIdx.x; j < kParts; j += kThreads) parts[j] = 0.0f;
}

template <int XT, int HT, int LPR, int CPT>
__global__ __launch_bounds__(Rows<LPR>::kThreads) void residual_norm_bwd_kernel(
    const void *__restrict__ dy, const u32x4 *__restrict__ dz, const void *__restrict__ x, const void *__restrict__ h,
    const float *__restrict__ weight, const float *__restrict__ post_weight, const float *__restrict__ gate, int gate_scalar, int64_t rows,
    int cols, float a, const float *__restrict__ stats, void *__restrict__ dx, void *__restrict__ dh, float *__restrict__ parts,
    float *__restrict__ slabs, float *__restrict__ gate_sums) {
    constexpr int kThreads = Rows<LPR>::kThreads, RPB = Rows<LPR>::kPerBlock;
    __shared__ float lds[2 * 3 * (LPR / kWave + 1)];
    __shared__ uint32_t red[kThreads / kWave];
    __shared__ float fold[RPB > 1 ? kThreads * 8 : 1];
    const int lane = threadIdx.x % LPR, nchunk = cols / 8;
    const int64_t step = (int64_t)gridDim.x * RPB;
    const float gs = gate && gate_scalar ? gate[0] : 1.0f;
    float wv[CPT][8], wn[CPT][8], dw[CPT][8], dd[CPT][8];
    double dg = 0.0;                                           // (a sum of everything, of both signs: held in 64 bits from row to row)
    lane_weights<CPT, LPR>(weight, post_weight, gate, gate_scalar, lane, nchunk, wv, wn);
#pragma unroll
    for (int j = 0; j < CPT; ++j)
#pragma unroll
        for (int e = 0; e < 8; ++e) dw[j][e] = dd[j][e] = 0.0f;

    u32x4 nx[CPT][kVecs<XT>], nh[CPT][kVecs<HT>], ny[CPT][kVecs<XT>], nz[CPT][1];
    float nrh = 1.0f, nry = 0.0f;
    auto fetch = [&](int64_t row) {
        const bool live = row < rows;
#pragma unroll
        for (int j = 0; j < CPT; ++j) {
            const int c = lane + j * LPR;
            const bool ok = live && c < nchunk;
            load8<XT>(x, row * nchunk + c, ok, nx[j]);
            load8<HT>(h, row * nchunk + c, ok, nh[j]);
            load8<XT>(dy, row * nchunk + c, ok && dy, ny[j]);
            load8<ODL_BF16>(dz, row * nchunk + c, ok && dz, nz[j]);
        }
        if (live) {
            nrh = stats[row];
            nry = stats[rows + row];
        }
    };
    int turn = 0;
    uint32_t am = 0;
    int64_t row = (int64_t)blockIdx.x * RPB + threadIdx.x / LPR;
    fetch(row);
    for (int64_t row0 = (int64_t)blockIdx.x * RPB; row0 < rows; row0 += step, row += step) {
        const float rh = nrh, ry = nry;
        float yf[CPT][8], hf[CPT][8], ef[CPT][8], zf[CPT][8];
#pragma unroll
        for (int j = 0; j < CPT; ++j) {
            widen8<XT>(nx[j], yf[j]);
            widen8<HT>(nh[j], hf[j]);
            widen8<XT>(ny[j], ef[j]);
            widen8<ODL_BF16>(nz[j], zf[j]);
        }
        fetch(row + step);
        float s[3] = {0.0f, 0.0f, 0.0f};                       // t * yh, k * (dy + ry * t), k * yh
#pragma unroll
        for (int j = 0; j < CPT; ++j)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                hf[j][e] *= rh;
                const float k = gs * wv[j][e] * hf[j][e];
                yf[j][e] = __fmaf_rn(a, yf[j][e], k) * ry;
                const float t = zf[j][e] * wn[j][e];
                dw[j][e] = __fmaf_rn(zf[j][e], yf[j][e], dw[j][e]);
                ef[j][e] = __fmaf_rn(ry, t, ef[j][e]);
                s[0] = __fmaf_rn(t, yf[j][e], s[0]);
                s[1] = __fmaf_rn(k, ef[j][e], s[1]);
                s[2] = __fmaf_rn(k, yf[j][e], s[2]);
            }
        row_sums<LPR, 3>(s, lds, turn);
        const float c2 = ry * (s[0] / (float)cols);
        float dg_row = 0.0f;
        const float c3 = post_weight ? __fmaf_rn(-c2, s[2], s[1]) / (float)cols : 0.0f;
        if (row < rows) {
#pragma unroll
            for (int j = 0; j < CPT; ++j) {
                const int c = lane + j * LPR;
                if (c < nchunk) {
                    float ox[8], oh[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const float ey = __fmaf_rn(-c2, yf[j][e], ef[j][e]);
                        const float eh = ey * hf[j][e];
                        dd[j][e] += eh;
                        dg_row = __fmaf_rn(eh, wv[j][e], dg_row);
                        ox[e] = a * ey;
                        oh[e] = rh * __fmaf_rn(-c3, hf[j][e], ey * (gs * wv[j][e]));
                    }
                    store8<XT>(dx, row * nchunk + c, ox);
                    store8<HT>(dh, row * nchunk + c, oh);
                    if constexpr (HT == ODL_BF16) {
#pragma unroll
                        for (int q = 0; q < 4; ++q) am = max_u16x2(am, abs_bf16x2(pack_bf16x2(oh[2 * q], oh[2 * q + 1])));
                    } else {
#pragma unroll
                        for (int e = 0; e < 8; ++e) am = max(am, float_to_bits(oh[e]) & 0x7fffffffu);
                    }
                }
            }
        }
        dg += dg_row;
    }
    if (parts) {
        am = block_max_u32(HT == ODL_BF16 ? fold_u16x2_to_f32bits(am) : am, red);
        if (threadIdx.x == 0) parts[blockIdx.x] = bits_to_float(am);
        if (blockIdx.x == 0)
            for (int j = (int)gridDim.x + threadIdx.x; j < kParts; j += kThreads) parts[j] = 0.0f;
    }
    if (!slabs) return;                                        // (uniform: none of the weights wants a gradient)

    // the block's sums of its columns as one slab: [d_weight, D]
    float *slab = slabs + (int64_t)blockIdx.x * 2 * cols;
    if constexpr (RPB == 1) {
#pragma unroll
        for (int j = 0; j < CPT; ++j) {
            const int c = lane + j * LPR;
            if (c < nchunk) {
                store8<ODL_F32>(slab, c, dw[j]);
                store8<ODL_F32>(slab + cols, c, dd[j]);
            }
        }
    } else {                                                   // the rows side by side in a block, in order
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
            for (int j = 0; j < CPT; ++j) {
                __syncthreads();
#pragma unroll
                for (int e = 0; e < 8; ++e) fold[e * kThreads + threadIdx.x] = half ? dd[j][e] : dw[j][e];
                __syncthreads();
                const int c = lane + j * LPR;
                if (threadIdx.x < LPR && c < nchunk) {
                    float s[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        s[e] = fold[e * kThreads + lane];
                        for (int r = 1; r < RPB; ++r) s[e] += fold[e * kThreads + r * LPR + lane];
                    }
                    store8<ODL_F32>(slab + half * cols, c, s);
                }
            }
    }
    if (gate_sums) {
        __shared__ double sums[kThreads / kWave];
#pragma unroll
        for (int off = kWave / 2; off > 0; off >>= 1) dg += __shfl_xor(dg, off, kWave);
        if (threadIdx.x % kWave == 0) sums[threadIdx.x / kWave] = dg;
        __syncthreads();
        if (threadIdx.x == 0) {
            double s = sums[0];
            for (int w = 1; w < kThreads / kWave; ++w) s += sums[w];
            gate_sums[blockIdx.x] = (float)s;
        }
    }
}

// Slabs [nslab][2 * cols] -> gradients of the weights.  A block owns 64 columns: 16 groups of lanes add every 16th slab, eight
// loads in flight, and are added up in group order.  The block behind the last columns adds up the scalar gate's sums.
__global__ __launch_bounds__(1024) void residual_norm_sums_kernel(const float *__restrict__ slabs, const float *__restrict__ gate_sums, int nslab,
                                                                  int cols, const float *__restrict__ post_weight,
                                                                  const float *__restrict__ gate, int gate_scalar, float *__restrict__ dweight,
                                                                  float *__restrict__ dpost, float *__restrict__ dgate) {
    __shared__ float part[16][64];
    const int cx = threadIdx.x % 64, grp = threadIdx.x / 64;
    if ((int)blockIdx.x == (2 * cols + 63) / 64) {
        if (grp == 0) {
            double a = 0.0;
            for (int b = cx; b < nslab; b += 64) a += gate_sums[b];
#pragma unroll
            for (int off = kWave / 2; off > 0; off >>= 1) a += __shfl_xor(a, off, kWave);
            if (cx == 0) dgate[0] = (float)a;
        }
        return;
    }
    const int c = (int)blockIdx.x * 64 + cx;
    float a = 0.0f;
    if (c < 2 * cols) {
        int b = grp;
        for (; b + 7 * 16 < nslab; b += 8 * 16) {
            float v[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) v[u] = slabs[(int64_t)(b + u * 16) * 2 * cols + c];
#pragma unroll
            for (int u = 0; u < 8; ++u) a += v[u];
        }
        for (; b < nslab; b += 16) a += slabs[(int64_t)b * 2 * cols + c];
    }
    part[grp][cx] = a;
    __syncthreads();
    if (grp != 0 || c >= 2 * cols) return;
    float t = part[0][cx];
#pragma unroll
    for (int g = 1; g < 16; ++g) t += part[g][cx];
    if (c < cols) {
        dweight[c] = t;
        return;
    }
    const int k = c - cols;
    if (dpost) dpost[k] = gate ? t * gate[gate_scalar ? 0 : k] : t;
    if (dgate && !gate_scalar) dgate[k] = post_weight ? t * post_weight[k] : t;
}

bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// lanes that hold a row
int lanes_of(int64_t cols) {
    return cols <= 128 ? 16 : cols <= 256 ? 32 : cols <= 1024 ? 64 : cols <= 4096 ? 256 : 512;
}

// A block for every partial maximum at most, two for every compute unit.
int64_t blocks_of(int64_t rows, int lanes) {
    const int64_t per = lanes > 256 ? 1 : 256 / lanes, want = (rows + per - 1) / per, cap = (int64_t)device_cu_count() * 2;
    const int64_t most = cap < kSlabs ? cap : kSlabs;
    return want < 1 ? 1 : want < most ? want : most;
}

int check_shape(const char *who, int x_dtype, int h_dtype, int64_t rows, int64_t cols, int64_t gate_size, const float *gate) {
    if (rows < 0 || cols < 0) return set_error(ODL_ERR_ARG, "%s: negative shape", who);
    if (!((x_dtype == ODL_BF16 && h_dtype == ODL_BF16) || (x_dtype == ODL_F32 && (h_dtype == ODL_BF16 || h_dtype == ODL_F32))))
        return set_error(ODL_ERR_ARG, "%s: x_dtype %d with h_dtype %d (h is bf16, or fp32 beside an fp32 x)", who, x_dtype, h_dtype);
    if (cols < 8 || cols % 8 != 0 || cols > 8192) return set_error(ODL_ERR_SHAPE, "%s: cols must be a multiple of 8 in [8, 8192]", who);
    if (gate && gate_size != 1 && gate_size != cols) return set_error(ODL_ERR_SHAPE, "%s: a gate has 1 or cols elements, not %lld", who, (long long)gate_size);
    return ODL_OK;
}

}  // namespace
}  // namespace odl

using namespace odl;

// one instance for each pair of types and row width
#define ODL_RN_TYPES(KERNEL, LPR, CPT)                                                                  \
    do {                                                                                                \
        if (x_dtype == ODL_BF16) ODL_RN_GO((KERNEL<ODL_BF16, ODL_BF16, LPR, CPT>), LPR);                \
        else if (h_dtype == ODL_BF16) ODL_RN_GO((KERNEL<ODL_F32, ODL_BF16, LPR, CPT>), LPR);            \
        else ODL_RN_GO((KERNEL<ODL_F32, ODL_F32, LPR, CPT>), LPR);                                      \
    } while (0)
#define ODL_RN_WIDTHS(KERNEL)                                                                           \
    do {                                                                                                \
        if (lanes == 16) ODL_RN_TYPES(KERNEL, 16, 1);                                                   \
        else if (lanes == 32) ODL_RN_TYPES(KERNEL, 32, 1);                                              \
        else if (lanes == 64 && cols <= 512) ODL_RN_TYPES(KERNEL, 64, 1);                               \
        else if (lanes == 64) ODL_RN_TYPES(KERNEL, 64, 2);                                              \
        else if (lanes == 256 && cols <= 2048) ODL_RN_TYPES(KERNEL, 256, 1);                            \
        else if (lanes == 256) ODL_RN_TYPES(KERNEL, 256, 2);                                            \
        else ODL_RN_TYPES(KERNEL, 512, 2);                                                              \
    } while (0)

extern "C" int odl_fp8_residual_norm(const void *x, int x_dtype, const void *h, int h_dtype, const float *weight, const float *post_weight,
                                     const float *gate, int64_t gate_size, int64_t rows, int64_t cols, float residual_scale, float eps,
                                     float post_eps, void *y, void *z, float *stats, float *parts, odl_stream_t stream_) {
    hipStream_t stream = reinterpret_cast<hipStream_t>(stream_);
    if (const int rc = check_shape("odl_fp8_residual_norm", x_dtype, h_dtype, rows, cols, gate_size, gate)) return rc;
    if (!weight || (rows > 0 && (!x || !h || !y || !z))) return set_error(ODL_ERR_ARG, "odl_fp8_residual_norm: null pointer");
    if (!aligned16(x) || !aligned16(h) || !aligned16(y) || !aligned16(z))
        return set_error(ODL_ERR_SHAPE, "odl_fp8_residual_norm: x, h, y and z must be 16-byte aligned");
    const int lanes = lanes_of(cols);
    const dim3 grid((unsigned)blocks_of(rows, lanes));
#define ODL_RN_GO(KERNEL, LPR)                                                                                                            \
    hipLaunchKernelGGL(KERNEL, grid, dim3(Rows<LPR>::kThreads), 0, stream, x, h, weight, post_weight, gate, (int)(gate_size == 1), rows, \
                       (int)cols, residual_scale, eps, post_eps, y, z, stats, parts)
    ODL_RN_WIDTHS(residual_norm_kernel);
#undef ODL_RN_GO
    return check_launch("odl_fp8_residual_norm");
}

extern "C" int odl_fp8_residual_norm_bwd(const void *dy, const void *dz, const void *x, int x_dtype, const void *h, int h_dtype, const float *weight,
                                         const float *post_weight, const float *gate, int64_t gate_size, int64_t rows, int64_t cols,
                                         float residual_scale, const float *stats, void *dx, void *dh, float *parts, float *dweight,
                                         float *dpost_weight, float *dgate, float *workspace, odl_stream_t stream_) {
    hipStream_t stream = reinterpret_cast<hipStream_t>(stream_);
    if (const int rc = check_shape("odl_fp8_residual_norm_bwd", x_dtype, h_dtype, rows, cols, gate_size, gate)) return rc;
    if (!weight || (rows > 0 && (!x || !h || !dx || !dh || !stats))) return set_error(ODL_ERR_ARG, "odl_fp8_residual_norm_bwd: null pointer");
    if (dweight && !workspace) return set_error(ODL_ERR_ARG, "odl_fp8_residual_norm_bwd: gradients of the weights need a workspace");
    if ((dpost_weight || dgate) && !dweight) return set_error(ODL_ERR_ARG, "odl_fp8_residual_norm_bwd: dweight comes with the other weights' gradients");
    if ((dpost_weight && !post_weight) || (dgate && !gate)) return set_error(ODL_ERR_ARG, "odl_fp8_residual_norm_bwd: a gradient of a weight that is not there");
    if (!aligned16(x) || !aligned16(h) || !aligned16(dy) || !aligned16(dz) || !aligned16(dx) || !aligned16(dh) || !aligned16(workspace))
        return set_error(ODL_ERR_SHAPE, "odl_fp8_residual_norm_bwd: the matrices and the workspace must be 16-byte aligned");
    const int lanes = lanes_of(cols), scalar = gate_size == 1;
    const int64_t blocks = blocks_of(rows, lanes);
    const dim3 grid((unsigned)blocks);
    float *slabs = dweight ? workspace : nullptr, *gate_sums = dgate && scalar ? workspace + 2 * kSlabs * cols : nullptr;
#define ODL_RN_GO(KERNEL, LPR)                                                                                                       \
    hipLaunchKernelGGL(KERNEL, grid, dim3(Rows<LPR>::kThreads), 0, stream, dy, reinterpret_cast<const u32x4 *>(dz), x, h, weight,    \
                       post_weight, gate, scalar, rows, (int)cols, residual_scale, stats, dx, dh, parts, slabs, gate_sums)
    ODL_RN_WIDTHS(residual_norm_bwd_kernel);
#undef ODL_RN_GO
    if (dweight)
        hipLaunchKernelGGL(residual_norm_sums_kernel, dim3((unsigned)((2 * cols + 63) / 64 + (gate_sums ? 1 : 0))), dim3(1024), 0, stream, slabs, gate_sums,
                           (int)blocks, (int)cols, post_weight, gate, scalar, dweight, dpost_weight, dgate);
    return check_launch("odl_fp8_residual_norm_bwd");
}
