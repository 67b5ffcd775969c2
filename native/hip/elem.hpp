// What the kernels that follow a reduction (norm.hip, adamw.hip) share: element types, wide loads
// and stores at any alignment, e4m3, reductions over a wavefront, and the device of a launch.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace netop {

enum Dtype : int { kF32 = 0, kBf16 = 1, kF16 = 2 };  // the codes of ops/hip.py:DTYPES

template <class T, int N>
using Vec = T __attribute__((ext_vector_type(N)));

// N elements at an address that is aligned to one element only.  global_load_dwordx4 and its like
// take any address (the HSA target runs in unaligned access mode), so rows of odd width and views
// at odd offsets use the same instructions as aligned ones.
template <class T, int N>
struct Wide {
    typedef Vec<T, N> Any __attribute__((aligned(sizeof(T))));
    __device__ static __forceinline__ Vec<T, N> load(const T* p) { return *reinterpret_cast<const Any*>(p); }
    __device__ static __forceinline__ Vec<T, N> stream(const T* p) {
        return __builtin_nontemporal_load(reinterpret_cast<const Any*>(p));
    }
    __device__ static __forceinline__ void store(T* p, const Vec<T, N>& v) { *reinterpret_cast<Any*>(p) = v; }
    __device__ static __forceinline__ void put(T* p, const Vec<T, N>& v) {
        __builtin_nontemporal_store(v, reinterpret_cast<Any*>(p));
    }
};

// To and from fp32; to 16 bits round to nearest even (v_cvt_pk_bf16_f32, v_cvt_f16_f32), NaN stays NaN.
template <class T, int N>
__device__ __forceinline__ Vec<float, N> widen(const Vec<T, N>& v) {
    return __builtin_convertvector(v, Vec<float, N>);
}
template <class T, int N>
__device__ __forceinline__ Vec<T, N> narrow(const Vec<float, N>& v) {
    return __builtin_convertvector(v, Vec<T, N>);
}

constexpr float kE4m3Max = 448.0f;
constexpr float kTiny = 0x1p-100f;  // values that share a scale and all lie below are stored as zeros

__device__ __forceinline__ float clamp_e4m3(float x) {  // NaN stays NaN
    return x > kE4m3Max ? kE4m3Max : x < -kE4m3Max ? -kE4m3Max : x;
}
// Four values within +-448 as e4m3 bytes, nearest even, lowest byte first.
__device__ __forceinline__ uint32_t pack_e4m3(float a, float b, float c, float d) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return uint32_t(__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true));
}
__device__ __forceinline__ Vec<float, 4> unpack_e4m3(uint32_t w) {
    const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8(int(w), false);
    const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8(int(w), true);
    return Vec<float, 4>{lo[0], lo[1], hi[0], hi[1]};
}

// Sums and maxima over WIDTH neighbouring lanes (a power of two up to 64); every lane gets the
// result, the same bits in each.
template <int WIDTH, class T>
__device__ __forceinline__ T lanes_sum(T x) {
#pragma unroll
    for (int m = 1; m < WIDTH; m <<= 1) x += __shfl_xor(x, m, 64);
    return x;
}
// Of non-negative values; a NaN wins when KEEP_NAN, else it is passed over.
template <int WIDTH, bool KEEP_NAN>
__device__ __forceinline__ float lanes_max(float x) {
#pragma unroll
    for (int m = 1; m < WIDTH; m <<= 1) {
        const float y = __shfl_xor(x, m, 64);
        x = KEEP_NAN ? (x > y || x != x ? x : y) : fmaxf(x, y);
    }
    return x;
}

// Launches run on the tensors' device, whichever device is current; the caller's comes back.
struct OnDevice {
    int prev = -1;
    hipError_t err;
    explicit OnDevice(int device) {
        err = hipGetDevice(&prev);
        if (err != hipSuccess || prev == device) {
            prev = -1;
            return;
        }
        const int was = prev;
        err = hipSetDevice(device);
        prev = err == hipSuccess ? was : -1;
    }
    ~OnDevice() {
        if (prev >= 0) (void)hipSetDevice(prev);
    }
    OnDevice(const OnDevice&) = delete;
    OnDevice& operator=(const OnDevice&) = delete;
};

}  // namespace netop
