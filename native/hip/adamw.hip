// The optimizer's side of a data-parallel step (gfx950): the global norm of the summed gradients
// and one AdamW step, each over many tensors at once.
//
//   g' = coef g
//   m  = b1 m + (1 - b1) g'            v = b2 v + (1 - b2) g'^2
//   p  = p (1 - lr wd) - lr (m / c1) / (sqrt(v / c2) + eps),   c1 = 1 - b1^step, c2 = 1 - b2^step
//
// All in fp32; 16-bit parameters are roundings of an fp32 master.  States take 32 bits, or 8: blocks
// of 256 elements of a tensor, which one wavefront holds, keep m and sqrt(v) as e4m3 codes times a
// scale (largest / 448).  The step uses the new m and v before they are rounded.  sqrt(v) is kept,
// not v: its range is half as many powers of two.
//
// The rounding is stochastic, from a hash of (seed, step, position): with b2 = 0.999 one step moves
// sqrt(v) by a hundredth of the distance of two codes, which rounding to nearest would lose every
// time, so that v would stand still.  A sqrt(v) other than zero never becomes zero: a zero below an
// m that is not would make the next update m / eps.
//
// Bound by HBM: with a bf16 gradient and parameter and an fp32 master 28 bytes an element, 16 with states in
// 8 bits.  2^29 elements of the one take 2.7 ms (5.6 TB/s, a large copy's rate), 2^28 of the other 0.74 ms
// (5.8 TB/s).  The 8-bit states' arithmetic comes near that too, some 100 instructions an element: before the
// bounds checks left whole chunks and the divisions the step it took 0.80 ms.
//
// What stochastic rounding costs: a value that moves by D times itself carries a noise of about the root
// of D / 10 (codes lie 6 to 12 % apart).  That is a tenth of m, which turns over in ten steps, and up to a
// third of sqrt(v) -- of each element on its own, around the right mean.
#include "elem.hpp"

#include <algorithm>

using namespace netop;

namespace {

constexpr int kThreads = 256;
constexpr int kBlock = 256;          // elements that share a scale: 64 lanes x 4
constexpr int kUnroll = 2;           // blocks a wavefront works on together: 4 leave uneven ends (2^28 elements: 4 % slower)
constexpr int kChunk = kThreads / 64 * kUnroll * kBlock;  // elements of one workgroup
constexpr int kMaxGrads = 440;       // gradient addresses that fit a launch's arguments (4 KiB)

// A workgroup's stretch of one tensor, in a table on the device (ops/adamw.py:AdamW).
struct Chunk {
    char* p;          // the parameter's first element here
    uint64_t offset;  // position in the flat states
    uint64_t start;   // first element within the tensor
    int32_t n;        // elements
    int32_t tensor;   // whose gradient: index into this launch's addresses
};

struct Hyper {
    float b1, one_b1, b2, one_b2, eps, decay, alpha, rc2;  // alpha = lr / c1, rc2 = 1 / sqrt(c2), decay = 1 - lr wd
    float scale;
    uint32_t key;
};

// As packed by ops/adamw.py:_STEP.
struct StepParams {
    const Chunk* chunks;
    float* master;       // flat; null where the parameters are fp32
    void* m;             // flat
    void* v;
    float* m_scale;      // per block; null with 32 bits
    float* v_scale;
    const float* coef;   // or null
    const Hyper* on_device;  // or null: where lr or step are tensors
    Hyper hyper;
    int32_t n_chunks, ptype, gtype, bits, n_grads, device;
};

struct Grads {
    const void* at[kMaxGrads];
};
static_assert(sizeof(StepParams) == 128 && sizeof(Hyper) == 40 && sizeof(Chunk) == 32, "ops/adamw.py packs these");
static_assert(sizeof(StepParams) + sizeof(Grads) <= 4096, "kernel arguments");

// Four random numbers, for the positions from a multiple of four on: one product reaches all of them.
// The two rounds of xor-shift and product are the 32-bit mixer of C. Wellons, "Prospecting for Hash
// Functions" (2018); the odd constants that spread position, seed and step come from the public-domain
// hashes of A. Appleby and Y. Collet, where any odd numbers of mixed bits would do.
__device__ __forceinline__ Vec<uint32_t, 4> random4(uint64_t position, uint32_t key) {
    constexpr uint32_t kLow = 0x9E3779B1u;
    const uint32_t low = uint32_t(position) * kLow, high = uint32_t(position >> 32) * 0x85EBCA77u ^ key;
    Vec<uint32_t, 4> r;
#pragma unroll
    for (uint32_t j = 0; j < 4; ++j) {
        uint32_t x = (low + j * kLow) ^ high;
        x ^= x >> 15;
        x *= 0x2C1B3C6Du;
        x ^= x >> 12;
        x *= 0x297A2D39u;
        r[j] = x ^ (x >> 15);
    }
    return r;
}

__host__ __device__ __forceinline__ uint32_t key_of(uint32_t seed, uint64_t step) {
    const uint32_t k = seed * 0x85EBCA6Bu + uint32_t(step) * 0xC2B2AE35u;
    return k ^ (k >> 16);
}

// u in [0, 448] as the code below or above it: above where its place between the two plus rnd / 2^16
// reaches one.  From 2^-6 on a code is the exponent and three bits of the fraction, so that adding the
// random number below those bits and cutting them off rounds; below, codes are multiples of 2^-9.
__device__ __forceinline__ uint32_t stochastic_e4m3(float u, uint32_t rnd) {
    const uint32_t normal = ((__float_as_uint(u) + (rnd << 4)) >> 20) - (120u << 3);
    const uint32_t small = uint32_t(fmaf(float(rnd), 0x1p-16f, u * 512.0f));
    return u < 0x1p-6f ? small : normal;
}

// n of four elements, zeros behind; all of them where the chunk is whole.
template <bool WHOLE, class T>
__device__ __forceinline__ Vec<float, 4> load4(const T* p, int n) {
    if (WHOLE || n >= 4) return widen<T, 4>(Wide<T, 4>::stream(p));
    Vec<float, 4> v = 0.0f;
#pragma unroll
    for (int j = 0; j < 3; ++j)
        if (j < n) v[j] = float(p[j]);
    return v;
}
template <bool WHOLE, class T>
__device__ __forceinline__ void store4(T* p, const Vec<float, 4>& v, int n) {
    if (WHOLE || n >= 4) {
        Wide<T, 4>::put(p, narrow<T, 4>(v));
        return;
    }
#pragma unroll
    for (int j = 0; j < 3; ++j)
        if (j < n) p[j] = T(v[j]);
}

// Products and sums are rounded one by one, not contracted: which way a state rounds hangs on the last
// bit, and is to follow from the formulas alone, whatever compiled them.  The quotient in p's step decides
// nothing and takes the hardware's reciprocal (1 ulp).
template <class P, class G, int BITS, bool WHOLE>
__device__ __forceinline__ void chunk_step(const StepParams& a, const Chunk& ch, const G* gp, const Hyper& hy, float coef) {
#pragma clang fp contract(off)
    constexpr bool kMaster = sizeof(P) == 2;
    P* pp = reinterpret_cast<P*>(ch.p);
    const int lane = threadIdx.x & 63;
    const int base = (threadIdx.x >> 6) * (kUnroll * kBlock) + lane * 4;
    Vec<float, 4> g[kUnroll], w[kUnroll], m[kUnroll], v[kUnroll];
    uint32_t mq[kUnroll], vq[kUnroll];
    float ms[kUnroll], vs[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
        const int i = base + u * kBlock, n = ch.n - i;
        if (!WHOLE && i - lane * 4 >= ch.n) break;  // the whole block lies behind the tensor's end
        const uint64_t at = ch.offset + i;
        g[u] = load4<WHOLE>(gp + i, n);
        w[u] = kMaster ? load4<WHOLE>(a.master + at, n) : load4<WHOLE>(reinterpret_cast<const float*>(pp) + i, n);
        if constexpr (BITS == 32) {  // states are padded to whole blocks
            m[u] = Wide<float, 4>::stream(static_cast<const float*>(a.m) + at);
            v[u] = Wide<float, 4>::stream(static_cast<const float*>(a.v) + at);
        } else {
            mq[u] = __builtin_nontemporal_load(reinterpret_cast<const uint32_t*>(static_cast<const char*>(a.m) + at));
            vq[u] = __builtin_nontemporal_load(reinterpret_cast<const uint32_t*>(static_cast<const char*>(a.v) + at));
            ms[u] = a.m_scale[at / kBlock];
            vs[u] = a.v_scale[at / kBlock];
        }
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
        const int i = base + u * kBlock, n = ch.n - i;
        if (!WHOLE && i - lane * 4 >= ch.n) break;
        const uint64_t at = ch.offset + i;
        if constexpr (BITS == 8) {
            m[u] = unpack_e4m3(mq[u]) * ms[u];
            v[u] = unpack_e4m3(vq[u]) * vs[u];
            v[u] *= v[u];
        }
        Vec<float, 4> root;
        float m_max = 0, r_max = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float x = g[u][j] * coef;
            m[u][j] = hy.b1 * m[u][j] + hy.one_b1 * x;
            v[u][j] = hy.b2 * v[u][j] + hy.one_b2 * (x * x);
            root[j] = sqrtf(v[u][j]);
            w[u][j] = w[u][j] * hy.decay - hy.alpha * m[u][j] * __builtin_amdgcn_rcpf(root[j] * hy.rc2 + hy.eps);
            m_max = fmaxf(m_max, fabsf(m[u][j]));
            r_max = fmaxf(r_max, root[j]);
        }
        if constexpr (kMaster) store4<WHOLE>(a.master + at, w[u], n);
        store4<WHOLE>(pp + i, w[u], n);
        if constexpr (BITS == 32) {
            Wide<float, 4>::put(static_cast<float*>(a.m) + at, m[u]);
            Wide<float, 4>::put(static_cast<float*>(a.v) + at, v[u]);
        } else {
            m_max = lanes_max<64, false>(m_max);
            r_max = lanes_max<64, false>(r_max);
            const float m_scale = m_max < kTiny ? 0.0f : m_max * (1.0f / kE4m3Max);
            const float r_scale = r_max < kTiny ? 0.0f : r_max * (1.0f / kE4m3Max);
            const float m_inv = m_max < kTiny ? 0.0f : 1.0f / m_scale;
            const float r_inv = r_max < kTiny ? 0.0f : 1.0f / r_scale;
            const Vec<uint32_t, 4> rnd = random4(at, hy.key);
            uint32_t mw = 0, vw = 0;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float x = m[u][j], r = root[j];
                uint32_t mc = stochastic_e4m3(fminf(fabsf(x) * m_inv, kE4m3Max), rnd[j] & 0xffffu);
                uint32_t vc = stochastic_e4m3(fminf(r * r_inv, kE4m3Max), rnd[j] >> 16);
                if (vc == 0 && r * r_inv > 0) vc = 1;
                mc = x != x ? 0x7fu : mc | (__float_as_uint(x) >> 24 & 0x80u);
                vc = r != r ? 0x7fu : vc;
                mw |= mc << (8 * j);
                vw |= vc << (8 * j);
            }
            __builtin_nontemporal_store(mw, reinterpret_cast<uint32_t*>(static_cast<char*>(a.m) + at));
            __builtin_nontemporal_store(vw, reinterpret_cast<uint32_t*>(static_cast<char*>(a.v) + at));
            if (lane == 0) {
                a.m_scale[at / kBlock] = m_scale;
                a.v_scale[at / kBlock] = r_scale;
            }
        }
    }
}

template <class P, class G, int BITS>
__global__ __launch_bounds__(kThreads) void adamw_kernel(StepParams a, Grads grads) {
    const Chunk ch = a.chunks[blockIdx.x];
    const G* gp = static_cast<const G*>(grads.at[ch.tensor]);
    if (!gp) return;  // no gradient: the tensor keeps its value and states
    const Hyper hy = a.on_device ? *a.on_device : a.hyper;
    float coef = hy.scale;
    if (a.coef) {
        coef *= *a.coef;
        if (!(fabsf(coef) < __builtin_inff())) return;  // the gradients overflowed: the step is left out
    }
    if (ch.n == kChunk)
        chunk_step<P, G, BITS, true>(a, ch, gp + ch.start, hy, coef);
    else
        chunk_step<P, G, BITS, false>(a, ch, gp + ch.start, hy, coef);
}

// The step's numbers where lr or step are on the device (a captured graph's are): 64 bits, since
// 1 - b^step cancels.
__global__ void hyper_kernel(Hyper* out, Hyper h, double b1, double b2, double lr, double decay, uint32_t seed,
                             const float* lr_dev, const int64_t* step_dev, int64_t step) {
    if (step_dev) step = *step_dev < 1 ? 1 : *step_dev;
    if (lr_dev) lr = double(*lr_dev);
    h.alpha = float(lr / -expm1(double(step) * log(b1)));
    h.rc2 = float(1.0 / sqrt(-expm1(double(step) * log(b2))));
    h.decay = float(1.0 - lr * decay);
    h.key = key_of(seed, uint64_t(step));
    *out = h;
}

template <class P, class G>
void launch_step(const StepParams& a, const Grads& g, hipStream_t stream) {
    if (a.bits == 8)
        hipLaunchKernelGGL((adamw_kernel<P, G, 8>), dim3(unsigned(a.n_chunks)), dim3(kThreads), 0, stream, a, g);
    else
        hipLaunchKernelGGL((adamw_kernel<P, G, 32>), dim3(unsigned(a.n_chunks)), dim3(kThreads), 0, stream, a, g);
}
template <class P>
bool launch_grads(const StepParams& a, const Grads& g, hipStream_t stream) {
    switch (a.gtype) {
        case kF32: launch_step<P, float>(a, g, stream); return true;
        case kBf16: launch_step<P, __bf16>(a, g, stream); return true;
        case kF16: launch_step<P, _Float16>(a, g, stream); return true;
        default: return false;
    }
}

// ---- the norm of many gradients -------------------------------------------------------------------
// Sums of squares in 64 bits throughout: squares of fp32 gradients leave fp32's range long before
// the gradients do, and 2^29 terms its precision.  A workgroup sums one stretch of one tensor; a
// second launch of one workgroup adds up the stretches in a fixed order.  Bound by HBM reads: 1 GiB of
// bf16 in 290 tensors takes 177 us (6.1 TB/s); 2^20 fp32 elements in 23 4.1 + 2.7 us, less than the host takes to
// ask for them.  Eight lanes add up a tensor's stretches, which a single large tensor waits for: 2^27 elements of one
// take 124 us, 2^24 49 us.
constexpr int kMaxNormTensors = 150;  // addresses and sizes that fit a launch's arguments
constexpr int kFinalThreads = 1024;

struct NormGroup {
    const void* at[kMaxNormTensors];
    uint64_t n[kMaxNormTensors];
    uint32_t first[kMaxNormTensors + 1];  // a tensor's first stretch
    int32_t tensors;
};
struct NormArgs {
    double* partial;   // a sum for each stretch of all groups, then one for each tensor
    double* per_tensor;
    float* norms;      // or null
    float* total;
    float* coef;       // or null
    float scale, max_norm;
    uint32_t base;     // the group's first stretch
    int32_t base_tensor, all_tensors, last;
    uint64_t stretch;
};
static_assert(sizeof(NormGroup) + sizeof(NormArgs) <= 4096, "kernel arguments");

template <class G>
__global__ __launch_bounds__(kThreads) void sumsq_kernel(NormGroup group, NormArgs a) {
    __shared__ double red[kThreads / 64];
    int lo = 0, hi = group.tensors - 1;  // the last tensor whose first stretch is not behind this one
    while (lo < hi) {
        const int mid = (lo + hi + 1) / 2;
        if (group.first[mid] <= blockIdx.x) lo = mid; else hi = mid - 1;
    }
    const uint64_t from = uint64_t(blockIdx.x - group.first[lo]) * a.stretch;
    const uint64_t left = group.n[lo] - from, n = left < a.stretch ? left : a.stretch;
    const G* p = static_cast<const G*>(group.at[lo]) + from;
    double s = 0;
    uint64_t i = uint64_t(threadIdx.x) * 8;
    constexpr uint64_t kStep = kThreads * 8;
    for (; i + 3 * kStep + 8 <= n; i += 4 * kStep) {  // four loads in flight a lane
        Vec<G, 8> v[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) v[u] = Wide<G, 8>::stream(p + i + u * kStep);
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
            for (int j = 0; j < 8; ++j) s = fma(double(float(v[u][j])), double(float(v[u][j])), s);
    }
    for (; i + 8 <= n; i += kStep) {
        const Vec<G, 8> v = Wide<G, 8>::load(p + i);
#pragma unroll
        for (int j = 0; j < 8; ++j) s = fma(double(float(v[j])), double(float(v[j])), s);
    }
    for (; i < n; ++i) s = fma(double(float(p[i])), double(float(p[i])), s);  // one thread's last elements
    s = lanes_sum<64>(s);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int k = 1; k < kThreads / 64; ++k) s += red[k];
        a.partial[a.base + blockIdx.x] = s;
    }
}

// Eight lanes a tensor add up its stretches; after the last group, all tensors' sums.
__global__ __launch_bounds__(kFinalThreads) void sumsq_final_kernel(NormGroup group, NormArgs a) {
    __shared__ double red[kFinalThreads / 64];
    for (int i0 = 0; i0 < group.tensors; i0 += kFinalThreads / 8) {
        const int i = i0 + int(threadIdx.x) / 8;
        double s = 0;
        if (i < group.tensors)
            for (uint32_t k = group.first[i] + (threadIdx.x & 7); k < group.first[i + 1]; k += 8) s += a.partial[a.base + k];
        s = lanes_sum<8>(s);
        if (i < group.tensors && (threadIdx.x & 7) == 0) {
            a.per_tensor[a.base_tensor + i] = s;
            if (a.norms) a.norms[a.base_tensor + i] = float(double(a.scale) * sqrt(s));
        }
    }
    if (!a.last) return;
    __syncthreads();  // this group's sums; earlier groups' are from launches before
    double s = 0;
    for (int i = threadIdx.x; i < a.all_tensors; i += kFinalThreads) s += a.per_tensor[i];
    s = lanes_sum<64>(s);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int k = 1; k < kFinalThreads / 64; ++k) s += red[k];
        const double total = double(a.scale) * sqrt(s);
        *a.total = float(total);
        if (a.coef) {
            const double clip = double(a.max_norm) / (total + 1e-6);
            *a.coef = float(double(a.scale) * (float(total) < __builtin_inff() ? (clip < 1 ? clip : 1.0) : __builtin_nan("")));
        }
    }
}

constexpr int kOverlap = -1;  // ops/adamw.py raises ValueError for it

// What a step writes, as packed by ops/adamw.py:_HELD: spans that do not overlap, by address.
struct Span {
    uint64_t from, to;
    int64_t owner;  // the parameter that it is, or -1
};
struct Held {
    const Span* spans;
    const uint64_t* elements;  // of each gradient
    int64_t n_spans, n;
};

// Whether a gradient (coef) lies in a span, except a gradient in its own parameter's, element on element.
bool strays(const Held& held, const void* const* grads, uint64_t size, uint64_t own_size, const float* coef) {
    const Span* end = held.spans + held.n_spans;
    for (int64_t i = 0; i <= held.n; ++i) {
        const bool is_coef = i == held.n;
        const auto at = reinterpret_cast<uintptr_t>(is_coef ? coef : grads[i]);
        const uint64_t bytes = is_coef ? 4 : held.elements[i] * size;
        if (!at || !bytes) continue;
        const Span* s = std::upper_bound(held.spans, end, uint64_t(at), [](uint64_t x, const Span& y) { return x < y.to; });
        if (s == end || s->from >= at + bytes) continue;  // the first that ends behind `at`
        if (is_coef || s->owner != i || s->from != at || size != own_size) return true;
    }
    return false;
}

}  // namespace

extern "C" {

// Return hipError_t values (0 = success), or -1 for tensors that may not share memory.

int netop_adamw_chunk() { return kChunk; }
int netop_adamw_max_grads() { return kMaxGrads; }
int netop_adamw_hyper_bytes() { return int(sizeof(Hyper)); }

// One launch over p->n_chunks chunks, whose tensors' gradients are grads[first .. first + n_grads).  With
// `held` every one of its n gradients and coef are looked up first: a gradient may lie where its own
// parameter does, element on element, and nowhere else that a step writes.
int netop_adamw_step(const StepParams* p, const void* const* grads, int first, const Held* held, hipStream_t stream) {
    if (!p || !grads || first < 0 || p->n_grads < 1 || p->n_grads > kMaxGrads || p->n_chunks < 0 || !p->m || !p->v ||
        (p->bits != 8 && p->bits != 32) || (p->bits == 8 && (!p->m_scale || !p->v_scale)) ||
        (p->ptype != kF32 && !p->master))
        return int(hipErrorInvalidValue);
    if (p->n_chunks == 0) return int(hipSuccess);
    // A grid's threads are counted in 32 bits.
    if (!p->chunks || uint64_t(p->n_chunks) * kThreads > 0xffffffffu) return int(hipErrorInvalidValue);
    if (held && strays(*held, grads, p->gtype == kF32 ? 4 : 2, p->ptype == kF32 ? 4 : 2, p->coef)) return kOverlap;
    const OnDevice on(p->device);
    if (on.err != hipSuccess) return int(on.err);
    Grads g;
    for (int i = 0; i < kMaxGrads; ++i) g.at[i] = i < p->n_grads ? grads[first + i] : nullptr;
    bool known = false;
    switch (p->ptype) {
        case kF32: known = launch_grads<float>(*p, g, stream); break;
        case kBf16: known = launch_grads<__bf16>(*p, g, stream); break;
        case kF16: known = launch_grads<_Float16>(*p, g, stream); break;
        default: break;
    }
    return known ? int(hipGetLastError()) : int(hipErrorInvalidValue);
}

// *out = the numbers of step *step_dev (or `step`) at learning rate *lr_dev (or `lr`).
int netop_adamw_hyper(void* out, const Hyper* h, double b1, double b2, double lr, double decay, uint32_t seed,
                      const float* lr_dev, const int64_t* step_dev, int64_t step, int device, hipStream_t stream) {
    if (!out || !h) return int(hipErrorInvalidValue);
    const OnDevice on(device);
    if (on.err != hipSuccess) return int(on.err);
    hipLaunchKernelGGL(hyper_kernel, dim3(1), dim3(1), 0, stream, static_cast<Hyper*>(out), *h, b1, b2, lr, decay, seed,
                       lr_dev, step_dev, step);
    return int(hipGetLastError());
}

// Elements that one workgroup sums: enough stretches to fill the chip, few enough to add up.
// `workspace` of netop_grad_norm: `stretches` doubles, at least ceil(n / stretch) a tensor, and one
// for each tensor.
int netop_grad_norm(const void* const* grads, const uint64_t* n, int tensors, int dtype, uint64_t stretch, void* workspace,
                    uint64_t stretches, float* total, float* norms, float* coef, float scale, float max_norm, int device,
                    hipStream_t stream) {
    if (!grads || !n || tensors < 1 || !workspace || !total || stretch < 1 || dtype < kF32 || dtype > kF16)
        return int(hipErrorInvalidValue);
    const struct {
        const void* at;
        uint64_t n;
    } outs[3] = {{total, 4}, {coef, 4}, {norms, uint64_t(tensors) * 4}};
    const auto meet = [](const void* a, uint64_t n, const void* b, uint64_t m) {
        const auto x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
        return x && y && n && m && x < y + m && y < x + n;
    };
    for (int i = 0; i < 3; ++i)
        for (int j = 0; j < i; ++j)
            if (meet(outs[i].at, outs[i].n, outs[j].at, outs[j].n)) return kOverlap;
    uint64_t need = 0;
    for (int i = 0; i < tensors; ++i) {
        if (n[i] && !grads[i]) return int(hipErrorInvalidValue);
        need += (n[i] + stretch - 1) / stretch;
        for (const auto& o : outs)  // a later group's gradients are read after this one's norms are written
            if (meet(o.at, o.n, grads[i], n[i] * (dtype == kF32 ? 4 : 2))) return kOverlap;
    }
    if (need > stretches || need * kThreads > 0xffffffffu) return int(hipErrorInvalidValue);
    const OnDevice on(device);
    if (on.err != hipSuccess) return int(on.err);
    NormArgs a{};
    a.partial = static_cast<double*>(workspace);
    a.per_tensor = a.partial + stretches;
    a.norms = norms;
    a.total = total;
    a.coef = coef;
    a.scale = scale;
    a.max_norm = max_norm;
    a.all_tensors = tensors;
    a.stretch = stretch;
    for (int t0 = 0; t0 < tensors; t0 += kMaxNormTensors) {
        NormGroup g{};
        g.tensors = tensors - t0 < kMaxNormTensors ? tensors - t0 : kMaxNormTensors;
        for (int i = 0; i < g.tensors; ++i) {
            g.at[i] = grads[t0 + i];
            g.n[i] = n[t0 + i];
            g.first[i + 1] = g.first[i] + uint32_t((n[t0 + i] + stretch - 1) / stretch);
        }
        a.base_tensor = t0;
        a.last = t0 + g.tensors == tensors;
        const unsigned blocks = g.first[g.tensors];
        if (blocks) {
            if (dtype == kF32)
                hipLaunchKernelGGL(sumsq_kernel<float>, dim3(blocks), dim3(kThreads), 0, stream, g, a);
            else if (dtype == kBf16)
                hipLaunchKernelGGL(sumsq_kernel<__bf16>, dim3(blocks), dim3(kThreads), 0, stream, g, a);
            else
                hipLaunchKernelGGL(sumsq_kernel<_Float16>, dim3(blocks), dim3(kThreads), 0, stream, g, a);
            const hipError_t e = hipGetLastError();
            if (e != hipSuccess) return int(e);
        }
        hipLaunchKernelGGL(sumsq_final_kernel, dim3(1), dim3(kFinalThreads), 0, stream, g, a);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return int(e);
        a.base += blocks;
    }
    return int(hipSuccess);
}

}  // extern "C"
