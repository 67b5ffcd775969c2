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
// One workgroup or one wavefront keeps a row of h in registers, so every input is read once and
// every output written once.  Bound by HBM; the arithmetic is about ten operations an element.
//
// Backward, with g = dy weight:  dh = rstd g - h rstd^3 mean(g h) + dresidual, which is the
// gradient of every partial sum and of the residual alike; dweight = sum over rows of dy h rstd.
#include "elem.hpp"

using namespace netop;

namespace {

constexpr int kMaxIn = 9;         // eight partial sums and the residual
constexpr int kMaxCols = 32768;   // a row in the registers of one workgroup
constexpr int kGroup = 128;       // columns that share a scale

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

// The sum of x over the TPR threads of a row, in every one of them.  `red`: TPR / 64 floats that
// the workgroup has not read since its last barrier.
template <int TPR>
__device__ __forceinline__ float row_sum(float x, float* red) {
    x = lanes_sum<64>(x);
    if constexpr (TPR > 64) {
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = x;
        __syncthreads();
        x = 0;
#pragma unroll
        for (int i = 0; i < TPR / 64; ++i) x += red[i];
    }
    return x;
}
template <int TPR>
__device__ __forceinline__ float row_max(float x, float* red) {
    x = lanes_max<64, true>(x);
    if constexpr (TPR > 64) {
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = x;
        __syncthreads();
        x = red[0];
#pragma unroll
        for (int i = 1; i < TPR / 64; ++i) x = x > red[i] || x != x ? x : red[i];
    }
    return x;
}

template <class T>
__device__ __forceinline__ Vec<float, 8> load8(const T* p, int n) {  // n < 8 elements, zeros behind
    Vec<float, 8> v = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; ++j)
        if (j < n) v[j] = float(p[j]);
    return v;
}

template <class T>
__device__ __forceinline__ Vec<float, 8> weights8(const void* w, int f32, int c, int n) {
    if (f32) {
        const float* p = static_cast<const float*>(w) + c;
        return n >= 8 ? Wide<float, 8>::load(p) : load8(p, n);
    }
    const T* p = static_cast<const T*>(w) + c;
    return n >= 8 ? widen<T, 8>(Wide<T, 8>::load(p)) : load8(p, n);
}

template <class T>
__device__ __forceinline__ void store8(T* p, const Vec<float, 8>& v, int n) {
    if (n >= 8) {
        Wide<T, 8>::store(p, narrow<T, 8>(v));
        return;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j)
        if (j < n) p[j] = T(v[j]);
}

// TPR threads hold a row, VPT vectors of 8 columns each: vector k of thread t is columns
// 8 (k TPR + t) and on.
template <class T, int TPR, int VPT, int OUT>
__global__ __launch_bounds__(TPR < 256 ? 256 : TPR) void norm_kernel(NormParams a) {
    constexpr int kRows = TPR < 256 ? 256 / TPR : 1;
    __shared__ float red[2][TPR / 64];
    const uint64_t row = uint64_t(blockIdx.x) * kRows + threadIdx.x / TPR;
    if (kRows > 1 && row >= a.rows) return;  // whole wavefronts: such rows meet no barrier
    const int t = threadIdx.x % TPR;
    const int cols = a.cols;
    Vec<float, 8> h[VPT];
#pragma unroll
    for (int k = 0; k < VPT; ++k) h[k] = 0.0f;
    // Loads of kAhead inputs are in flight together: with peer pointers each is an xGMI round trip.
    constexpr int kAhead = 8 / VPT > 0 ? 8 / VPT : 1;
    for (int s0 = 0; s0 < a.n_in; s0 += kAhead) {
        Vec<T, 8> v[kAhead][VPT];
#pragma unroll
        for (int s = 0; s < kAhead; ++s) {
            if (s0 + s >= a.n_in) break;
            const T* p = static_cast<const T*>(a.in[s0 + s]) + int64_t(row) * a.in_stride[s0 + s];
#pragma unroll
            for (int k = 0; k < VPT; ++k) {
                const int c = (k * TPR + t) * 8;
                if (c + 8 <= cols) v[s][k] = Wide<T, 8>::load(p + c);
            }
        }
#pragma unroll
        for (int s = 0; s < kAhead; ++s) {
            if (s0 + s >= a.n_in) break;
#pragma unroll
            for (int k = 0; k < VPT; ++k) {
                const int c = (k * TPR + t) * 8;
                if (c + 8 <= cols) {
                    h[k] += widen<T, 8>(v[s][k]);
                } else if (c < cols) {
                    const T* p = static_cast<const T*>(a.in[s0 + s]) + int64_t(row) * a.in_stride[s0 + s];
                    h[k] += load8(p + c, cols - c);
                }
            }
        }
    }
    float ss = 0;
#pragma unroll
    for (int k = 0; k < VPT; ++k)
#pragma unroll
        for (int j = 0; j < 8; ++j) ss = fmaf(h[k][j], h[k][j], ss);
    ss = row_sum<TPR>(ss, red[0]);
    const float rstd = 1.0f / sqrtf(ss / float(cols) + a.eps);
    if (a.rstd && t == 0) a.rstd[row] = rstd;
    if (a.h) {  // after the reduction: every thread of the row has read its inputs, which h may replace
        T* p = static_cast<T*>(a.h) + int64_t(row) * a.h_stride;
#pragma unroll
        for (int k = 0; k < VPT; ++k) {
            const int c = (k * TPR + t) * 8;
            if (c < cols) store8(p + c, h[k], cols - c);
        }
    }
    float amax = 0;
#pragma unroll
    for (int k = 0; k < VPT; ++k) {
        const int c = (k * TPR + t) * 8;
        if (c < cols) h[k] = h[k] * rstd * weights8<T>(a.weight, a.weight_f32, c, cols - c);
        if constexpr (OUT == kRowScale) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float y = fabsf(h[k][j]);
                amax = amax > y || amax != amax ? amax : y;
            }
        }
    }
    if constexpr (OUT == kSame) {
        T* p = static_cast<T*>(a.out) + int64_t(row) * a.out_stride;
#pragma unroll
        for (int k = 0; k < VPT; ++k) {
            const int c = (k * TPR + t) * 8;
            if (c < cols) store8(p + c, h[k], cols - c);
        }
    } else {
        uint8_t* p = static_cast<uint8_t*>(a.out) + int64_t(row) * a.out_stride;
        if constexpr (OUT == kRowScale) {
            amax = row_max<TPR>(amax, red[1]);
            if (t == 0) a.scales[row] = amax < kTiny ? 0.0f : amax / kE4m3Max;
        }
        const int groups = (cols + kGroup - 1) / kGroup;
#pragma unroll
        for (int k = 0; k < VPT; ++k) {
            const int c = (k * TPR + t) * 8;
            if constexpr (OUT == kGroupScale) {  // 16 neighbouring threads hold a group
                amax = 0;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float y = fabsf(h[k][j]);
                    amax = amax > y || amax != amax ? amax : y;
                }
                amax = lanes_max<16, true>(amax);
                if ((t & 15) == 0 && c < cols) a.scales[row * groups + c / kGroup] = amax < kTiny ? 0.0f : amax / kE4m3Max;
            }
            const float inv = amax < kTiny ? 0.0f : kE4m3Max / amax;
            if (c < cols) {
                Vec<float, 8> q;
#pragma unroll
                for (int j = 0; j < 8; ++j) q[j] = clamp_e4m3(h[k][j] * inv);
                Vec<uint32_t, 2> w;
                w[0] = pack_e4m3(q[0], q[1], q[2], q[3]);
                w[1] = pack_e4m3(q[4], q[5], q[6], q[7]);
                if (cols - c >= 8) {
                    const auto bytes = __builtin_bit_cast(decltype(Vec<uint8_t, 8>()), w);
                    Wide<uint8_t, 8>::store(p + c, bytes);
                } else {
#pragma unroll
                    for (int j = 0; j < 7; ++j)
                        if (j < cols - c) p[c + j] = uint8_t(w[j >> 2] >> (8 * (j & 3)));
                }
            }
        }
    }
}

// Each row's share of dweight stays in the registers of the thread that holds those columns; a
// workgroup walks rows in steps of the grid and writes one partial row in the end, which
// dweight_kernel adds up in a fixed order: no atomics, the same bits every time.
template <class T, int TPR, int VPT>
__global__ __launch_bounds__(TPR < 256 ? 256 : TPR) void norm_backward_kernel(NormBackwardParams a) {
    constexpr int kRows = TPR < 256 ? 256 / TPR : 1;
    __shared__ float red[2][TPR / 64];
    const int part = int(blockIdx.x) * kRows + int(threadIdx.x) / TPR;
    if (kRows > 1 && part >= a.parts) return;  // whole wavefronts, as above
    const int t = threadIdx.x % TPR;
    const int cols = a.cols;
    Vec<float, 8> dw[VPT];
#pragma unroll
    for (int k = 0; k < VPT; ++k) dw[k] = 0.0f;
    int turn = 0;
    for (uint64_t row = part; row < a.rows; row += a.parts, turn ^= 1) {
        const T* dy = static_cast<const T*>(a.dy) + int64_t(row) * a.dy_stride;
        const T* hp = static_cast<const T*>(a.h) + int64_t(row) * a.h_stride;
        const float rstd = a.rstd[row];
        Vec<float, 8> g[VPT], h[VPT];
        float dot = 0;
#pragma unroll
        for (int k = 0; k < VPT; ++k) {
            const int c = (k * TPR + t) * 8;
            g[k] = h[k] = 0.0f;
            if (c + 8 <= cols) {
                g[k] = widen<T, 8>(Wide<T, 8>::load(dy + c));
                h[k] = widen<T, 8>(Wide<T, 8>::load(hp + c));
            } else if (c < cols) {
                g[k] = load8(dy + c, cols - c);
                h[k] = load8(hp + c, cols - c);
            }
        }
#pragma unroll
        for (int k = 0; k < VPT; ++k) {
            const int c = (k * TPR + t) * 8;
            dw[k] += g[k] * h[k] * rstd;
            if (c < cols) g[k] *= weights8<T>(a.weight, a.weight_f32, c, cols - c);
#pragma unroll
            for (int j = 0; j < 8; ++j) dot = fmaf(g[k][j], h[k][j], dot);
        }
        dot = row_sum<TPR>(dot, red[turn]);
        const float back = rstd * rstd * rstd * (dot / float(cols));
        T* dh = static_cast<T*>(a.dh) + int64_t(row) * a.dh_stride;
        const T* dres = static_cast<const T*>(a.dres) + (a.dres ? int64_t(row) * a.dres_stride : 0);
#pragma unroll
        for (int k = 0; k < VPT; ++k) {
            const int c = (k * TPR + t) * 8;
            if (c >= cols) continue;
            Vec<float, 8> d = rstd * g[k] - h[k] * back;
            if (a.dres) d += cols - c >= 8 ? widen<T, 8>(Wide<T, 8>::load(dres + c)) : load8(dres + c, cols - c);
            store8(dh + c, d, cols - c);
        }
    }
#pragma unroll
    for (int k = 0; k < VPT; ++k) {
        const int c = (k * TPR + t) * 8;
        if (c < cols) store8(a.partial + uint64_t(part) * cols + c, dw[k], cols - c);
    }
}

// dweight[c] = sum of partial[.][c]: 32 columns x 32 strands of parts a workgroup.
__global__ __launch_bounds__(1024) void dweight_kernel(const float* __restrict__ partial, int parts, int cols,
                                                       void* __restrict__ dweight, int dtype) {
    __shared__ float sum[32][33];
    const int x = threadIdx.x & 31, y = threadIdx.x >> 5;
    const int c = blockIdx.x * 32 + x;
    float s = 0;
    if (c < cols)
        for (int p = y; p < parts; p += 32) s += partial[uint64_t(p) * cols + c];
    sum[y][x] = s;
    __syncthreads();
    if (y == 0 && c < cols) {
        s = 0;
#pragma unroll
        for (int i = 0; i < 32; ++i) s += sum[i][x];
        if (dtype == kF32)
            static_cast<float*>(dweight)[c] = s;
        else if (dtype == kBf16)
            static_cast<__bf16*>(dweight)[c] = __bf16(s);
        else
            static_cast<_Float16*>(dweight)[c] = _Float16(s);
    }
}

// ---- which threads hold a row -------------------------------------------------------------------
struct Shape {
    int tpr, vpt;
};

Shape shape_for(int cols) {
    const int vecs = (cols + 7) / 8;
    if (vecs <= 64) return {64, 1};
    if (vecs <= 128) return {64, 2};
    if (vecs <= 256) return {256, 1};
    if (vecs <= 512) return {256, 2};
    if (vecs <= 1024) return {256, 4};
    if (vecs <= 2048) return {1024, 2};
    return {1024, 4};
}

template <class T, int TPR, int VPT>
void launch_norm(const NormParams& a, hipStream_t stream) {
    constexpr int kRows = TPR < 256 ? 256 / TPR : 1;
    const dim3 grid(unsigned((a.rows + kRows - 1) / kRows)), block(TPR < 256 ? 256 : TPR);
    if (a.out_kind == kSame)
        hipLaunchKernelGGL((norm_kernel<T, TPR, VPT, kSame>), grid, block, 0, stream, a);
    else if (a.out_kind == kRowScale)
        hipLaunchKernelGGL((norm_kernel<T, TPR, VPT, kRowScale>), grid, block, 0, stream, a);
    else
        hipLaunchKernelGGL((norm_kernel<T, TPR, VPT, kGroupScale>), grid, block, 0, stream, a);
}

template <class T, int TPR, int VPT>
void launch_backward(const NormBackwardParams& a, hipStream_t stream) {
    constexpr int kRows = TPR < 256 ? 256 / TPR : 1;
    hipLaunchKernelGGL((norm_backward_kernel<T, TPR, VPT>), dim3(unsigned((a.parts + kRows - 1) / kRows)),
                       dim3(TPR < 256 ? 256 : TPR), 0, stream, a);
}

#define NETOP_FOR_SHAPE(s, CALL)                         \
    do {                                                 \
        if (s.tpr == 64 && s.vpt == 1) CALL(64, 1);      \
        else if (s.tpr == 64) CALL(64, 2);               \
        else if (s.tpr == 256 && s.vpt == 1) CALL(256, 1); \
        else if (s.tpr == 256 && s.vpt == 2) CALL(256, 2); \
        else if (s.tpr == 256) CALL(256, 4);             \
        else if (s.vpt == 2) CALL(1024, 2);              \
        else CALL(1024, 4);                              \
    } while (0)

template <class T>
void norm_of(const NormParams& a, hipStream_t stream) {
    const Shape s = shape_for(a.cols);
#define CALL(TPR, VPT) launch_norm<T, TPR, VPT>(a, stream)
    NETOP_FOR_SHAPE(s, CALL);
#undef CALL
}
template <class T>
void backward_of(const NormBackwardParams& a, hipStream_t stream) {
    const Shape s = shape_for(a.cols);
#define CALL(TPR, VPT) launch_backward<T, TPR, VPT>(a, stream)
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
    switch (p->dtype) {
        case kF32: norm_of<float>(*p, stream); break;
        case kBf16: norm_of<__bf16>(*p, stream); break;
        case kF16: norm_of<_Float16>(*p, stream); break;
        default: return int(hipErrorInvalidValue);
    }
    return int(hipGetLastError());
}

// How many rows of `cols` floats the backward pass needs as workspace.
int netop_norm_backward_parts(uint64_t rows, int cols) {
    if (cols < 1 || cols > kMaxCols) return 0;
    const uint64_t most = shape_for(cols).tpr == 64 ? 4096 : 1024;
    return int(rows < most ? rows : most);
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
    hipLaunchKernelGGL(dweight_kernel, dim3(unsigned(p->cols + 31) / 32), dim3(1024), 0, stream, p->partial, p->parts,
                       p->cols, p->dweight, p->dweight_f32 ? int(kF32) : p->dtype);
    return int(hipGetLastError());
}

}  // extern "C"
