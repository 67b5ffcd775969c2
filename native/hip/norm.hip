// Residual RMS norm over partial sums (gfx950): what follows the sum of a tensor-parallel layer.
//
//   h = sum_k src_k + residual          fp32, in list order, the residual last
//   residual_out = round(h)             the stream's type, nearest even
//   rstd = 1 / sqrt(mean(h^2) + eps)
//   y = h rstd weight                   from the unrounded h; rounded once, to the stream's type
//                                       or to e4m3 with a scale a row / a scale each 128 columns
//
// The n = 1..8 partial sums may be peer memory (the one-shot all-reduce of xgmi_comm.py reads
// every rank's partials in place), so no sum is written before it is normalised.
//
// A row of h stays in the registers of a workgroup, or of a part of a wavefront, so every input is read
// once and every output written once.  Bound by HBM, the arithmetic is about ten operations an element:
// 16384 x 8192 bf16 with a residual to e4m3 takes 172 us (5.5 TB/s, a large copy's rate), 8192 x 4096 fp32 97 us.
// Few rows are bound by the way there and back: 64 x 8192 over 8 partial sums 5.8 us, one row of 4096 2.7 us.
//
// Backward, with x = h rstd and g = dy weight:  dh = rstd (g - x mean(g x)) + dresidual, which is the
// gradient of every partial sum and of the residual alike; dweight = sum over rows of dy x.  x is of
// order one whatever h is; rstd^3 would leave fp32 for rows of 1e13 or 1e-13, and dy h for others.
// 8192 x 4096 bf16 takes 44 us and 5 us for dweight (5.5 TB/s); where rows are few and wide, one workgroup a CU
// and the partial rows of dweight bound it: 333 x 10007 fp32 13 + 5 us, at 7 us of data.  Beyond 16384 columns,
// registers do: 3000 x 20000 bf16 135 us, at 86 us of data.
#include "elem.hpp"

using namespace netop;

namespace {

constexpr int kMaxIn = 9;         // eight partial sums and the residual
constexpr int kMaxCols = 32768;   // a row in the registers of one workgroup
constexpr int kGroup = 128;       // columns that share a scale
constexpr uint64_t kMaxRows = 1 << 21;  // of a launch: rows x 1024 threads stay below 2^32, the most a grid may have

enum Out : int { kSame = 0, kRowScale = 1, kGroupScale = 2 };

// As packed by ops/norm.py:_FORWARD.  Strides in elements.
struct NormParams {
    const void* in[kMaxIn];
    int64_t in_stride[kMaxIn];
    const void* weight;
    void* out;
    int64_t out_stride;
    void* h;  // or null
    int64_t h_stride;
    float* rstd;    // or null
    float* scales;  // or null
    uint64_t rows;
    int32_t cols, n_in, dtype, weight_f32, out_kind, device;
    float eps;
    int32_t pad;
};

// As packed by ops/norm.py:_BACKWARD.
struct NormBackwardParams {
    const void* dy;
    int64_t dy_stride;
    const void* h;
    int64_t h_stride;
    const void* dres;  // or null
    int64_t dres_stride;
    const void* weight;
    const float* rstd;
    void* dh;
    int64_t dh_stride;
    void* dweight;
    float* partial;  // [parts, cols]
    uint64_t rows;
    int32_t cols, parts, dtype, weight_f32, dweight_f32, device;
};
static_assert(sizeof(NormParams) == 240 && sizeof(NormBackwardParams) == 128, "ops/norm.py packs these");

// A row's threads: TPR of them, several rows a workgroup, or (TPR = 0) the whole workgroup, whose size
// then follows from the width: no wavefront idles because a width is no power of two.
template <int TPR>
struct Threads {
    static constexpr int kBlock = TPR ? 256 : 1024;  // at most
    static constexpr int kRows = TPR ? 256 / TPR : 1;
    static constexpr bool kAlone = TPR && TPR <= 64;  // a row lies within a wavefront: no barriers
    static constexpr int kSlots = TPR ? 4 : 16;       // wavefronts of a workgroup
    __device__ static __forceinline__ int per_row() { return TPR ? TPR : int(blockDim.x); }
    __device__ static __forceinline__ int mine() { return TPR ? int(threadIdx.x) % TPR : int(threadIdx.x); }
    __device__ static __forceinline__ int row() { return TPR ? int(threadIdx.x) / TPR : 0; }
};

// The sum (the maximum) of x over a row's threads, in every one of them.  `red`: a float for each
// wavefront of the workgroup, which nobody has read since the last barrier.
template <int TPR>
__device__ __forceinline__ float row_sum(float x, float* red) {
    using Th = Threads<TPR>;
    x = lanes_sum<(Th::kAlone ? TPR : 64)>(x);
    if constexpr (!Th::kAlone) {
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = x;
        __syncthreads();
        const int waves = Th::per_row() / 64, first = Th::row() * waves, i = threadIdx.x & 15;
        x = lanes_sum<16>(i < waves ? red[first + i] : 0.0f);
    }
    return x;
}
template <int TPR>
__device__ __forceinline__ float row_max(float x, float* red) {
    using Th = Threads<TPR>;
    x = lanes_max<(Th::kAlone ? TPR : 64), true>(x);
    if constexpr (!Th::kAlone) {
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = x;
        __syncthreads();
        const int waves = Th::per_row() / 64, first = Th::row() * waves, i = threadIdx.x & 15;
        x = lanes_max<16, true>(i < waves ? red[first + i] : 0.0f);
    }
    return x;
}

// Vectors of a row.  Its n threads hold VPT vectors of 8 columns each: vector k of thread t is columns
// 8 (k n + t) and on.  One that would end behind the row is the row's last eight columns instead: every
// load and store stays one instruction without a branch, columns that two threads hold come out the same
// in both, and sums count them once (`twice` columns are left out).  Taking such a vector element by
// element made a row of 5004 columns a third slower than one of 5008.  Rows have 8 columns at least.
// WHOLE: the width is a multiple of eight, and none of this arises.
template <bool WHOLE>
struct At {
    int c, twice;
    bool in;
    __device__ __forceinline__ At(int vec, int cols) : in(vec * 8 < cols) {
        c = WHOLE || vec * 8 + 8 <= cols ? vec * 8 : cols - 8;
        twice = WHOLE ? 0 : vec * 8 - c;
    }
};

template <class T, int VPT, bool WHOLE, bool STREAM>
struct Row {
    Vec<T, 8> v[VPT];
    __device__ __forceinline__ void load(const T* p, int t, int n, int cols) {
#pragma unroll
        for (int k = 0; k < VPT; ++k) {
            const At<WHOLE> at(k * n + t, cols);
            if (at.in) v[k] = STREAM ? Wide<T, 8>::stream(p + at.c) : Wide<T, 8>::load(p + at.c);
        }
    }
};

__device__ __forceinline__ float dot8(const Vec<float, 8>& x, const Vec<float, 8>& y, int twice, float s) {
    if (twice) {
#pragma unroll
        for (int j = 1; j < 8; ++j) s = fmaf(j >= twice ? x[j] : 0.0f, y[j], s);
        return s;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) s = fmaf(x[j], y[j], s);
    return s;
}

template <class T>
__device__ __forceinline__ Vec<float, 8> weights8(const void* w, int f32, int c) {
    return f32 ? Wide<float, 8>::load(static_cast<const float*>(w) + c)
               : widen<T, 8>(Wide<T, 8>::load(static_cast<const T*>(w) + c));
}

// The larger of two magnitudes; NaN stays.
__device__ __forceinline__ float larger(float x, float y) { return x > y || x != x ? x : y; }

// What values up to amax are stored with, and the factor of their codes: the reciprocal of the scale as it
// is stored, so that code x scale is nearest by that scale.
__device__ __forceinline__ void scale_of(float amax, float& scale, float& inv) {
    scale = amax < kTiny ? 0.0f : amax / kE4m3Max;
    inv = amax < kTiny ? 0.0f : 1.0f / scale;
}

// AHEAD inputs are on their way together: with peer pointers each is an xGMI round trip.
template <class T, int TPR, int VPT, int AHEAD, bool E4M3, bool WHOLE, bool STREAM>
__global__ __launch_bounds__(Threads<TPR>::kBlock) void norm_kernel(NormParams a) {
    using Th = Threads<TPR>;
    __shared__ float red[2][Th::kSlots];
    const uint64_t row = uint64_t(blockIdx.x) * Th::kRows + Th::row();
    const bool here = row < a.rows;
    if (Th::kAlone && !here) return;  // all threads of the row
    const int t = Th::mine(), n = Th::per_row();
    const int cols = here ? a.cols : 0;
    Vec<float, 8> h[VPT];
#pragma unroll
    for (int k = 0; k < VPT; ++k) h[k] = 0.0f;
    for (int s0 = 0; s0 < a.n_in; s0 += AHEAD) {
        Row<T, VPT, WHOLE, STREAM> in[AHEAD];
#pragma unroll
        for (int s = 0; s < AHEAD; ++s)
            if (s0 + s < a.n_in) in[s].load(static_cast<const T*>(a.in[s0 + s]) + int64_t(row) * a.in_stride[s0 + s], t, n, cols);
#pragma unroll
        for (int s = 0; s < AHEAD; ++s)
            if (s0 + s < a.n_in) {
#pragma unroll
                for (int k = 0; k < VPT; ++k)
                    if (At<WHOLE>(k * n + t, cols).in) h[k] += widen<T, 8>(in[s].v[k]);
            }
    }
    float ss = 0;
#pragma unroll
    for (int k = 0; k < VPT; ++k) {
        const At<WHOLE> at(k * n + t, cols);
        if (at.in) ss = dot8(h[k], h[k], at.twice, ss);
    }
    ss = row_sum<TPR>(ss, red[0]);
    const float rstd = 1.0f / sqrtf(ss / float(a.cols) + a.eps);
    if (a.rstd && t == 0 && here) a.rstd[row] = rstd;
    if (a.h) {  // after the reduction: every thread of the row has read its inputs, which h may replace
        T* p = static_cast<T*>(a.h) + int64_t(row) * a.h_stride;
#pragma unroll
        for (int k = 0; k < VPT; ++k) {
            const At<WHOLE> at(k * n + t, cols);
            if (at.in) Wide<T, 8>::store(p + at.c, narrow<T, 8>(h[k]));
        }
    }
    float amax = 0;
#pragma unroll
    for (int k = 0; k < VPT; ++k) {
        const At<WHOLE> at(k * n + t, cols);
        if (at.in) h[k] = h[k] * rstd * weights8<T>(a.weight, a.weight_f32, at.c);
        if constexpr (E4M3) {
#pragma unroll
            for (int j = 0; j < 8; ++j) amax = larger(amax, fabsf(h[k][j]));
        }
    }
    if constexpr (!E4M3) {
        T* p = static_cast<T*>(a.out) + int64_t(row) * a.out_stride;
#pragma unroll
        for (int k = 0; k < VPT; ++k) {
            const At<WHOLE> at(k * n + t, cols);
            if (at.in) Wide<T, 8>::store(p + at.c, narrow<T, 8>(h[k]));
        }
    } else {
        uint8_t* p = static_cast<uint8_t*>(a.out) + int64_t(row) * a.out_stride;
        const bool by_group = a.out_kind == kGroupScale;
        const int groups = (cols + kGroup - 1) / kGroup;
        float scale = 0, inv = 0;
        if (!by_group) {
            amax = row_max<TPR>(amax, red[1]);
            scale_of(amax, scale, inv);
            if (t == 0 && here) a.scales[row] = scale;
        }
#pragma unroll
        for (int k = 0; k < VPT; ++k) {
            const At<WHOLE> at(k * n + t, cols);
            if (by_group) {  // 16 neighbouring threads hold a group
                amax = 0;
#pragma unroll
                for (int j = 0; j < 8; ++j) amax = j >= at.twice ? larger(amax, fabsf(h[k][j])) : amax;
                amax = lanes_max<(TPR == 8 ? 8 : 16), true>(amax);
                scale_of(amax, scale, inv);
                if ((t & 15) == 0 && at.in) a.scales[row * groups + (k * n + t) / 16] = scale;
            }
            if (!at.in) continue;
            Vec<float, 8> q;
#pragma unroll
            for (int j = 0; j < 8; ++j) q[j] = clamp_e4m3(h[k][j] * inv);
            Vec<uint32_t, 2> w;
            w[0] = pack_e4m3(q[0], q[1], q[2], q[3]);
            w[1] = pack_e4m3(q[4], q[5], q[6], q[7]);
            if (by_group && at.twice) {  // its first columns may be of the group before, with another scale
#pragma unroll
                for (int j = 1; j < 8; ++j)
                    if (j >= at.twice) p[at.c + j] = uint8_t(w[j >> 2] >> (8 * (j & 3)));
            } else {
                const auto bytes = __builtin_bit_cast(decltype(Vec<uint8_t, 8>()), w);
                Wide<uint8_t, 8>::store(p + at.c, bytes);
            }
        }
    }
}

// Rows of less than eight columns: a thread each.
template <class T>
__global__ __launch_bounds__(256) void narrow_norm_kernel(NormParams a) {
    const uint64_t row = uint64_t(blockIdx.x) * 256 + threadIdx.x;
    if (row >= a.rows) return;
    float h[7], y[7], ss = 0, amax = 0;
#pragma unroll
    for (int c = 0; c < 7; ++c) h[c] = y[c] = 0;
    for (int s = 0; s < a.n_in; ++s) {
        const T* p = static_cast<const T*>(a.in[s]) + int64_t(row) * a.in_stride[s];
#pragma unroll
        for (int c = 0; c < 7; ++c)
            if (c < a.cols) h[c] += float(p[c]);
    }
#pragma unroll
    for (int c = 0; c < 7; ++c) ss = fmaf(h[c], h[c], ss);
    const float rstd = 1.0f / sqrtf(ss / float(a.cols) + a.eps);
    if (a.rstd) a.rstd[row] = rstd;
#pragma unroll
    for (int c = 0; c < 7; ++c)
        if (c < a.cols) {
            if (a.h) (static_cast<T*>(a.h) + int64_t(row) * a.h_stride)[c] = T(h[c]);
            y[c] = h[c] * rstd * (a.weight_f32 ? static_cast<const float*>(a.weight)[c] : float(static_cast<const T*>(a.weight)[c]));
            amax = larger(amax, fabsf(y[c]));
        }
    float scale, inv;
    scale_of(amax, scale, inv);
    if (a.out_kind != kSame) a.scales[row] = scale;
#pragma unroll
    for (int c = 0; c < 7; ++c)
        if (c < a.cols) {
            if (a.out_kind == kSame)
                (static_cast<T*>(a.out) + int64_t(row) * a.out_stride)[c] = T(y[c]);
            else
                (static_cast<uint8_t*>(a.out) + int64_t(row) * a.out_stride)[c] =
                    uint8_t(pack_e4m3(clamp_e4m3(y[c] * inv), 0, 0, 0));
        }
}

// Each row's share of dweight stays in the registers of the thread that holds those columns; a
// workgroup walks rows in steps of the grid, adds up its rows' shares and writes one partial row,
// and dweight_kernel adds those up: a fixed order, no atomics, the same bits every time.  With four
// vectors of fp32 a thread 128 registers do not hold a row beside dweight, and it is read a second time, out
// of the caches.  (Fetching the next row ahead costs as many registers and gained nothing: 53 against 51 us
// at 8192 x 4096.)
template <class T, int TPR, int VPT, bool WHOLE, bool STREAM>
__global__ __launch_bounds__(Threads<TPR>::kBlock) void norm_backward_kernel(NormBackwardParams a) {
    using Th = Threads<TPR>;
    constexpr int kRows = Th::kRows;
    constexpr bool kTwice = VPT == 4 && sizeof(T) == 4, kWeights = VPT <= 2;
    __shared__ float red[2][Th::kSlots];
    const int t = Th::mine(), n = Th::per_row(), r = Th::row();
    const uint64_t first = uint64_t(blockIdx.x) * kRows, walk = uint64_t(gridDim.x) * kRows;
    Vec<float, 8> dw[VPT], weight[VPT];
#pragma unroll
    for (int k = 0; k < VPT; ++k) {
        dw[k] = 0.0f;
        const At<WHOLE> at(k * n + t, a.cols);
        if (kWeights && at.in) weight[k] = weights8<T>(a.weight, a.weight_f32, at.c);
    }
    int turn = 0;
    // Rows that share barriers take as many turns as the workgroup's first.
    for (uint64_t base = first, row = first + r; (Th::kAlone ? row : base) < a.rows; base += walk, row += walk, turn ^= 1) {
        const int cols = row < a.rows ? a.cols : 0;
        const float rstd = cols ? a.rstd[row] : 0.0f;
        const T* dy = static_cast<const T*>(a.dy) + int64_t(row) * a.dy_stride;
        const T* hp = static_cast<const T*>(a.h) + int64_t(row) * a.h_stride;
        const T* rp = a.dres ? static_cast<const T*>(a.dres) + int64_t(row) * a.dres_stride : nullptr;
        T* dh = static_cast<T*>(a.dh) + int64_t(row) * a.dh_stride;
        Row<T, VPT, WHOLE, STREAM> raw_g, raw_h, raw_r;
        if constexpr (!kTwice) {
            raw_g.load(dy, t, n, cols);
            raw_h.load(hp, t, n, cols);
            if (rp) raw_r.load(rp, t, n, cols);
        }
        float dot = 0;
#pragma unroll
        for (int k = 0; k < VPT; ++k) {
            const At<WHOLE> at(k * n + t, cols);
            if (at.in) {
                if constexpr (kTwice) {
                    raw_g.v[k] = Wide<T, 8>::load(dy + at.c);
                    raw_h.v[k] = Wide<T, 8>::load(hp + at.c);
                }
                if constexpr (!kWeights) weight[k] = weights8<T>(a.weight, a.weight_f32, at.c);
                const Vec<float, 8> g = widen<T, 8>(raw_g.v[k]), x = widen<T, 8>(raw_h.v[k]) * rstd;
                dw[k] += g * x;
                dot = dot8(g * weight[k], x, at.twice, dot);
            }
            if constexpr (!kWeights) asm volatile("" ::: "memory");  // holds back the next vector's loads
        }
        dot = row_sum<TPR>(dot, red[turn]);
        const float back = dot / float(a.cols);
        Vec<T, 8> d[VPT];
#pragma unroll
        for (int k = 0; k < VPT; ++k) {
            const At<WHOLE> at(k * n + t, cols);
            if (at.in) {
                if constexpr (kTwice) {
                    raw_g.v[k] = Wide<T, 8>::load(dy + at.c);
                    raw_h.v[k] = Wide<T, 8>::load(hp + at.c);
                    if (rp) raw_r.v[k] = Wide<T, 8>::load(rp + at.c);
                }
                if constexpr (!kWeights) weight[k] = weights8<T>(a.weight, a.weight_f32, at.c);
                const Vec<float, 8> x = widen<T, 8>(raw_h.v[k]) * rstd;
                Vec<float, 8> y = rstd * (widen<T, 8>(raw_g.v[k]) * weight[k] - x * back);
                if (rp) y += widen<T, 8>(raw_r.v[k]);
                d[k] = narrow<T, 8>(y);
                if constexpr (!kTwice) Wide<T, 8>::store(dh + at.c, d[k]);
            }
            if constexpr (!kWeights) asm volatile("" ::: "memory");
        }
        if constexpr (kTwice) {
            __syncthreads();  // dh may be where two threads have just read the same columns
#pragma unroll
            for (int k = 0; k < VPT; ++k) {
                const At<WHOLE> at(k * n + t, cols);
                if (at.in) Wide<T, 8>::store(dh + at.c, d[k]);
            }
        }
    }
    if constexpr (kRows > 1) {
        __shared__ Vec<float, 8> shares[kRows][TPR];
        shares[r][t] = dw[0];
        __syncthreads();
        if (r) return;
#pragma unroll
        for (int i = 1; i < kRows; ++i) dw[0] += shares[i][t];
    }
#pragma unroll
    for (int k = 0; k < VPT; ++k) {
        const At<WHOLE> at(k * n + t, a.cols);
        if (at.in) Wide<float, 8>::store(a.partial + uint64_t(blockIdx.x) * a.cols + at.c, dw[k]);
    }
}

template <class T>
__global__ __launch_bounds__(256) void narrow_backward_kernel(NormBackwardParams a) {
    __shared__ float shares[4][7];
    float dw[7], w[7];
#pragma unroll
    for (int c = 0; c < 7; ++c) {
        dw[c] = w[c] = 0;
        if (c < a.cols) w[c] = a.weight_f32 ? static_cast<const float*>(a.weight)[c] : float(static_cast<const T*>(a.weight)[c]);
    }
    for (uint64_t row = uint64_t(blockIdx.x) * 256 + threadIdx.x; row < a.rows; row += uint64_t(gridDim.x) * 256) {
        const T* dy = static_cast<const T*>(a.dy) + int64_t(row) * a.dy_stride;
        const T* hp = static_cast<const T*>(a.h) + int64_t(row) * a.h_stride;
        const T* rp = a.dres ? static_cast<const T*>(a.dres) + int64_t(row) * a.dres_stride : nullptr;
        T* dh = static_cast<T*>(a.dh) + int64_t(row) * a.dh_stride;
        const float rstd = a.rstd[row];
        float g[7], x[7], dot = 0;
#pragma unroll
        for (int c = 0; c < 7; ++c) {
            g[c] = x[c] = 0;
            if (c < a.cols) {
                g[c] = float(dy[c]);
                x[c] = float(hp[c]) * rstd;
            }
            dw[c] += g[c] * x[c];
            g[c] *= w[c];
            dot = fmaf(g[c], x[c], dot);
        }
        const float back = dot / float(a.cols);
#pragma unroll
        for (int c = 0; c < 7; ++c)
            if (c < a.cols) dh[c] = T(rstd * (g[c] - x[c] * back) + (rp ? float(rp[c]) : 0.0f));
    }
#pragma unroll
    for (int c = 0; c < 7; ++c) {
        dw[c] = lanes_sum<64>(dw[c]);
        if ((threadIdx.x & 63) == 0) shares[threadIdx.x >> 6][c] = dw[c];
    }
    __syncthreads();
    const int c = threadIdx.x;
    if (c < a.cols)
        a.partial[uint64_t(blockIdx.x) * a.cols + c] = shares[0][c] + shares[1][c] + shares[2][c] + shares[3][c];
}

// dweight[c] = sum of partial[.][c]: 64 columns (16 lanes x 4) and 64 strands of parts a workgroup.
__global__ __launch_bounds__(1024) void dweight_kernel(const float* __restrict__ partial, int parts, int cols,
                                                       void* __restrict__ dweight, int dtype) {
    __shared__ float sum[16][64];
    const int x = threadIdx.x & 15, y = threadIdx.x >> 4;
    const int c = blockIdx.x * 64 + x * 4;
    Vec<float, 4> s = 0.0f;
    if (c + 4 <= cols) {
        int p = y;
        for (; p + 192 < parts; p += 256) {  // four loads in flight
            Vec<float, 4> v[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) v[u] = Wide<float, 4>::load(partial + uint64_t(p + 64 * u) * cols + c);
#pragma unroll
            for (int u = 0; u < 4; ++u) s += v[u];
        }
        for (; p < parts; p += 64) s += Wide<float, 4>::load(partial + uint64_t(p) * cols + c);
    } else if (c < cols) {
        for (int p = y; p < parts; p += 64)
#pragma unroll
            for (int j = 0; j < 3; ++j)
                if (c + j < cols) s[j] += partial[uint64_t(p) * cols + c + j];
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {  // the four strands of a wavefront, then the sixteen wavefronts
        s[j] += __shfl_xor(s[j], 16, 64);
        s[j] += __shfl_xor(s[j], 32, 64);
        if ((threadIdx.x & 48) == 0) sum[threadIdx.x >> 6][x * 4 + j] = s[j];
    }
    __syncthreads();
    const int i = threadIdx.x, at = blockIdx.x * 64 + i;
    if (i < 64 && at < cols) {
        float all = 0;
#pragma unroll
        for (int w = 0; w < 16; ++w) all += sum[w][i];
        if (dtype == kF32)
            static_cast<float*>(dweight)[at] = all;
        else if (dtype == kBf16)
            static_cast<__bf16*>(dweight)[at] = __bf16(all);
        else
            static_cast<_Float16*>(dweight)[at] = _Float16(all);
    }
}

// ---- which threads hold a row -------------------------------------------------------------------
struct Shape {
    int tpr, vpt, block;
};

// One vector a thread up to 4096 columns: fewest registers, most rows in flight.  Beyond, rows of two
// vectors a thread leave each CU more workgroups (16384 x 8192 bf16 to e4m3: 176 us with 512 threads, 202 with
// 1024), while few rows end sooner spread wider.  Of calls of 64, 300, 700 and 1001 rows with 1024 / 512 threads:
// 8192 bf16 over 8 partial sums 11.1 / 11.3, 11.5 / 11.6, 20.9 / 21.7 and 27.7 / 28.6 us, backward of 300, 700 and
// 1001 x 5003 12.1 / 12.9, 16.0 / 17.6 and 17.8 / 20.1.  Wider loses where a second round of rows is short:
// 1001 x 8192 of one source 13.3 / 11.5 us, 1001 x 5003 of three 12.4 / 11.7.
Shape shape_for(int cols, uint64_t rows) {
    const int vecs = (cols + 7) / 8;
    for (int tpr = 8; tpr <= 128; tpr *= 2)
        if (vecs <= tpr) return {tpr, 1, 256};
    const int vpt = vecs <= 512 || (vecs <= 1024 && rows <= 1024) ? 1 : vecs <= 2048 ? 2 : 4;
    // Four vectors a thread need every wavefront there is room for (backward 3000 x 20000: 135 us, 198 with 640).
    return {0, vpt, vpt == 4 ? 1024 : ((vecs + vpt - 1) / vpt + 63) / 64 * 64};
}

// Workgroups of the backward pass, each with a partial row of dweight: as many as are at work together, and
// few where rows are few, since a partial row costs two rows of fp32.  8192 x 4096 bf16: 512 50 us, 256 66,
// 1024 57; 8192 x 7168 fp32: 256 172 us, 512 182; 1000 x 5003 bf16: 256 17.4 us, 512 21.7; 65536 x 1024 bf16
// (two rows a workgroup): 768 96 us, 512 109, 1024 99.
int parts_for(int cols, uint64_t rows) {
    const Shape s = shape_for(cols, rows);
    const uint64_t at_once = cols < 8 ? 256 : s.tpr ? 256 / s.tpr : 1;
    const uint64_t most = cols < 8 || s.tpr ? 768 : rows >= 2048 && s.vpt == 1 && s.block <= 640 ? 512 : 256;
    const uint64_t need = (rows + at_once - 1) / at_once, turns = (need + most - 1) / most;
    return turns ? int((need + turns - 1) / turns) : 0;  // all of them as many turns: 333 rows are 167 times two
}

// Inputs of 64 MiB and more are read past the caches: they hardly lie there (256 MB) and will not be read
// again.  4096 x 4096 bf16 28.1 -> 25.7 us, backward 8192 x 4096 54 -> 51; inputs that do lie there are slower
// that way (1001 x 5003, 3 partial sums: 15.0 -> 17.7).  Not fp32, whose vectors are two loads of half lines.
bool past_caches(uint64_t rows, int cols, int inputs) {
    return rows * uint64_t(cols) * uint64_t(inputs) * 2 >= 64u << 20;
}

template <class T, int TPR, int VPT>
void launch_norm(const NormParams& a, int block, hipStream_t stream) {
    constexpr int kRows = Threads<TPR>::kRows, kMany = 8 / VPT > 2 ? 8 / VPT : 2;
    const dim3 grid(unsigned((a.rows + kRows - 1) / kRows));
    const bool few = a.n_in <= 2, whole = a.cols % 8 == 0, eight = a.out_kind != kSame;
    constexpr bool kStreams = sizeof(T) == 2;
    const bool streams = kStreams && past_caches(a.rows, a.cols, a.n_in);
    const auto k = !whole    ? eight ? norm_kernel<T, TPR, VPT, 2, true, false, false> : norm_kernel<T, TPR, VPT, 2, false, false, false>
                   : !few    ? eight ? norm_kernel<T, TPR, VPT, kMany, true, true, false> : norm_kernel<T, TPR, VPT, kMany, false, true, false>
                   : streams ? eight ? norm_kernel<T, TPR, VPT, 2, true, true, kStreams> : norm_kernel<T, TPR, VPT, 2, false, true, kStreams>
                   : eight   ? norm_kernel<T, TPR, VPT, 2, true, true, false>
                             : norm_kernel<T, TPR, VPT, 2, false, true, false>;
    hipLaunchKernelGGL(k, grid, dim3(unsigned(block)), 0, stream, a);
}

template <class T, int TPR, int VPT>
void launch_backward(const NormBackwardParams& a, int block, hipStream_t stream) {
    constexpr bool kStreams = sizeof(T) == 2;
    const auto k = a.cols % 8 ? norm_backward_kernel<T, TPR, VPT, false, false>
                   : kStreams && past_caches(a.rows, a.cols, a.dres ? 3 : 2) ? norm_backward_kernel<T, TPR, VPT, true, kStreams>
                                                                            : norm_backward_kernel<T, TPR, VPT, true, false>;
    hipLaunchKernelGGL(k, dim3(unsigned(a.parts)), dim3(unsigned(block)), 0, stream, a);
}

#define NETOP_FOR_SHAPE(s, CALL)              \
    do {                                      \
        switch (s.tpr) {                      \
            case 8: CALL(8, 1); break;        \
            case 16: CALL(16, 1); break;      \
            case 32: CALL(32, 1); break;      \
            case 64: CALL(64, 1); break;      \
            case 128: CALL(128, 1); break;    \
            default:                          \
                if (s.vpt == 1) CALL(0, 1);   \
                else if (s.vpt == 2) CALL(0, 2); \
                else CALL(0, 4);              \
        }                                     \
    } while (0)

template <class T>
void norm_of(const NormParams& a, hipStream_t stream) {
    if (a.cols < 8) {
        hipLaunchKernelGGL(narrow_norm_kernel<T>, dim3(unsigned((a.rows + 255) / 256)), dim3(256), 0, stream, a);
        return;
    }
    const Shape s = shape_for(a.cols, a.rows);
#define CALL(TPR, VPT) launch_norm<T, TPR, VPT>(a, s.block, stream)
    NETOP_FOR_SHAPE(s, CALL);
#undef CALL
}
template <class T>
void backward_of(const NormBackwardParams& a, hipStream_t stream) {
    if (a.cols < 8) {
        hipLaunchKernelGGL(narrow_backward_kernel<T>, dim3(unsigned(a.parts)), dim3(256), 0, stream, a);
        return;
    }
    const Shape s = shape_for(a.cols, a.rows);
#define CALL(TPR, VPT) launch_backward<T, TPR, VPT>(a, s.block, stream)
    NETOP_FOR_SHAPE(s, CALL);
#undef CALL
}

// ---- memory that one call may not use twice ------------------------------------------------------
struct Span {
    uintptr_t at;
    uint64_t rows, pitch, width;  // bytes
};
uint64_t size_of(int dtype) { return dtype == kF32 ? 4 : 2; }

Span span(const void* p, uint64_t rows, int64_t stride, uint64_t cols, uint64_t size) {
    return {reinterpret_cast<uintptr_t>(p), rows, uint64_t(stride) * size, cols * size};
}

// Whether two spans share a byte.  Rows of one pitch may lie side by side (columns of one buffer).
bool meet(const Span& a, const Span& b) {
    if (!a.at || !b.at || !a.rows || !b.rows) return false;
    const uintptr_t ae = a.at + (a.rows - 1) * a.pitch + a.width, be = b.at + (b.rows - 1) * b.pitch + b.width;
    if (ae <= b.at || be <= a.at) return false;
    if (a.pitch == b.pitch && a.pitch) {
        const Span& lo = a.at <= b.at ? a : b;
        const Span& hi = a.at <= b.at ? b : a;
        const uint64_t d = (hi.at - lo.at) % a.pitch;
        if (d >= lo.width && d + hi.width <= a.pitch) return false;
    }
    return true;
}
bool same(const Span& a, const Span& b) {
    return a.at == b.at && a.width == b.width && (a.rows <= 1 || a.pitch == b.pitch);
}

constexpr int kOverlap = -1;  // ops/norm.py raises ValueError for it

}  // namespace

extern "C" {

// Returns a hipError_t value (0 = success), or -1 where an output overlaps an input in another way
// than element on element, or another output.  Nothing but the launch happens on the stream.
int netop_add_rms_norm(const NormParams* p, hipStream_t stream) {
    if (!p || p->n_in < 1 || p->n_in > kMaxIn || p->cols < 1 || p->cols > kMaxCols || p->rows > 0x7fffffffu ||
        !p->weight || !p->out || p->out_kind < kSame || p->out_kind > kGroupScale || (p->out_kind != kSame && !p->scales))
        return int(hipErrorInvalidValue);
    if (p->rows == 0) return int(hipSuccess);
    const uint64_t es = size_of(p->dtype), rows = p->rows, cols = uint64_t(p->cols);
    const uint64_t groups = p->out_kind == kGroupScale ? (cols + kGroup - 1) / kGroup : 1;
    const Span outs[4] = {span(p->out, rows, p->out_stride, cols, p->out_kind == kSame ? es : 1),
                          span(p->h, rows, p->h_stride, cols, es), span(p->rstd, rows, 1, 1, 4),
                          span(p->scales, rows, int64_t(groups), groups, 4)};
    const Span weight = span(p->weight, 1, 0, cols, p->weight_f32 ? 4 : es);
    for (int i = 0; i < 4; ++i) {
        for (int j = 0; j < i; ++j)
            if (meet(outs[i], outs[j])) return kOverlap;
        if (meet(outs[i], weight)) return kOverlap;
        for (int k = 0; k < p->n_in; ++k) {
            const Span in = span(p->in[k], rows, p->in_stride[k], cols, es);
            if (!in.at) return int(hipErrorInvalidValue);
            if (meet(outs[i], in) && !(i < 2 && same(outs[i], in))) return kOverlap;
        }
    }
    const OnDevice on(p->device);
    if (on.err != hipSuccess) return int(on.err);
    const auto moved = [](auto* q, int64_t bytes) { return q ? static_cast<decltype(q)>(static_cast<void*>(
        const_cast<char*>(static_cast<const char*>(static_cast<const void*>(q))) + bytes)) : q; };
    for (uint64_t r = 0; r < rows; r += kMaxRows) {
        NormParams a = *p;
        const int64_t at = int64_t(r);
        a.rows = rows - r < kMaxRows ? rows - r : kMaxRows;
        for (int k = 0; k < a.n_in; ++k) a.in[k] = moved(a.in[k], at * a.in_stride[k] * int64_t(es));
        a.out = moved(a.out, at * a.out_stride * (a.out_kind == kSame ? int64_t(es) : 1));
        a.h = moved(a.h, at * a.h_stride * int64_t(es));
        a.rstd = moved(a.rstd, at * 4);
        a.scales = moved(a.scales, at * int64_t(groups) * 4);
        switch (a.dtype) {
            case kF32: norm_of<float>(a, stream); break;
            case kBf16: norm_of<__bf16>(a, stream); break;
            case kF16: norm_of<_Float16>(a, stream); break;
            default: return int(hipErrorInvalidValue);
        }
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return int(e);
    }
    return int(hipSuccess);
}

// How many rows of `cols` floats the backward pass needs as workspace.
int netop_norm_backward_parts(uint64_t rows, int cols) {
    if (cols < 1 || cols > kMaxCols) return 0;
    return parts_for(cols, rows);
}

int netop_add_rms_norm_backward(const NormBackwardParams* p, hipStream_t stream) {
    if (!p || p->cols < 1 || p->cols > kMaxCols || p->rows > 0x7fffffffu || !p->weight || !p->dweight ||
        p->parts != netop_norm_backward_parts(p->rows, p->cols) ||
        (p->rows && (!p->dy || !p->h || !p->rstd || !p->dh || !p->partial)))
        return int(hipErrorInvalidValue);
    const uint64_t es = size_of(p->dtype), rows = p->rows, cols = uint64_t(p->cols);
    const Span dh = span(p->dh, rows, p->dh_stride, cols, es);
    const Span dw = span(p->dweight, 1, 0, cols, p->dweight_f32 ? 4 : es);
    const Span weight = span(p->weight, 1, 0, cols, p->weight_f32 ? 4 : es), rstd = span(p->rstd, rows, 1, 1, 4);
    const Span ins[3] = {span(p->dy, rows, p->dy_stride, cols, es), span(p->h, rows, p->h_stride, cols, es),
                         span(p->dres, rows, p->dres_stride, cols, es)};
    if (meet(dh, dw) || meet(dh, weight) || meet(dh, rstd) || meet(dw, weight) || meet(dw, rstd)) return kOverlap;
    for (const Span& in : ins)
        if ((meet(dh, in) && !same(dh, in)) || meet(dw, in)) return kOverlap;
    const OnDevice on(p->device);
    if (on.err != hipSuccess) return int(on.err);
    if (p->rows) {
        switch (p->dtype) {
            case kF32: backward_of<float>(*p, stream); break;
            case kBf16: backward_of<__bf16>(*p, stream); break;
            case kF16: backward_of<_Float16>(*p, stream); break;
            default: return int(hipErrorInvalidValue);
        }
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return int(e);
    }
    hipLaunchKernelGGL(dweight_kernel, dim3(unsigned(p->cols + 63) / 64), dim3(1024), 0, stream, p->partial, p->parts,
                       p->cols, p->dweight, p->dweight_f32 ? int(kF32) : p->dtype);
    return int(hipGetLastError());
}

}  // extern "C"
