// Shared by the sequence operators (norm.hip, convolution.hip, scan.hip, sample.hip): argument checks
// and the few device helpers they have in common.
#pragma once

#include "common.h"

namespace cnh {

// The library's device made current for a call on a thread that has another one selected (a caller
// that drives several devices), and the thread's own device restored afterwards.
class DeviceScope {
public:
    int enter() {
        CNH_HIP(hipGetDevice(&prev_));
        if (prev_ != current_device()) {
            CNH_HIP(hipSetDevice(current_device()));
            changed_ = true;
        }
        return 0;
    }
    ~DeviceScope() {
        if (changed_)
            (void)hipSetDevice(prev_);
    }

private:
    int prev_ = 0;
    bool changed_ = false;
};

// Elements from the first to the last of outer x inner rows of `cols` elements (0 when there are
// none), -1 when a stride is negative or the sum leaves 62 bits.
inline int64_t span_of(int64_t outer, int64_t outer_stride, int64_t inner, int64_t inner_stride, int64_t cols) {
    if (outer < 1 || inner < 1 || cols < 1)
        return 0;
    if (outer_stride < 0 || inner_stride < 0)
        return -1;
    __int128 n = (__int128)(outer - 1) * outer_stride + (__int128)(inner - 1) * inner_stride + cols;
    return n >= ((__int128)1 << 59) ? -1 : (int64_t)n;
}

// Are the rows of an output apart from each other, whichever of the two dimensions is the outer one
// in memory?
inline bool rows_apart(int64_t outer, int64_t outer_stride, int64_t inner, int64_t inner_stride, int64_t cols) {
    if (outer <= 1)
        return inner <= 1 || inner_stride >= cols;
    if (inner <= 1)
        return outer_stride >= cols;
    const bool outer_is_big = outer_stride >= inner_stride;
    const int64_t small = outer_is_big ? inner_stride : outer_stride, n = outer_is_big ? inner : outer;
    const int64_t big = outer_is_big ? outer_stride : inner_stride;
    return small >= cols && (__int128)big >= (__int128)(n - 1) * small + cols;
}

// One operand of a call, from its first byte to its last, for the overlap checks.
struct Extent {
    const char* what;
    const void* ptr;
    int64_t bytes;
};
inline bool overlap(const Extent& a, const Extent& b) {
    if (!a.ptr || !b.ptr || a.bytes <= 0 || b.bytes <= 0)
        return false;
    const uintptr_t pa = (uintptr_t)a.ptr, pb = (uintptr_t)b.ptr;
    return pa < pb + (uintptr_t)b.bytes && pb < pa + (uintptr_t)a.bytes;
}

inline bool aligned_to(const void* p, size_t n);
inline int check_extent(const Extent& e, int esz, const char* call) {
    CNH_CHECK(!e.ptr || e.bytes >= 0, -2, "%s: a stride of %s is negative or too large", call, e.what);
    CNH_CHECK(aligned_to(e.ptr, (size_t)esz), -2, "%s: %s is not aligned to its elements", call, e.what);
    return 0;
}

inline bool aligned_to(const void* p, size_t n) { return ((uintptr_t)p & (n - 1)) == 0; }

inline int check_float_type(int dtype, const char* call) {
    CNH_CHECK(dtype == CNH_F32 || dtype == CNH_F64, -2, "%s: element type %d is not fp32 or fp64", call, dtype);
    return 0;
}

// 16 bytes of elements, the widest access a lane makes.
template <typename T>
struct Wide;
template <>
struct Wide<float> {
    typedef float type __attribute__((ext_vector_type(4)));
    static constexpr int n = 4;
};
template <>
struct Wide<double> {
    typedef double type __attribute__((ext_vector_type(2)));
    static constexpr int n = 2;
};

// VEC consecutive elements in registers, moved as 16-byte accesses when VEC is Wide<T>::n or a multiple.
template <typename T, int VEC>
struct Pack {
    T v[VEC];
};
template <typename T, int VEC>
__device__ __forceinline__ void load_pack(Pack<T, VEC>& p, const T* at) {
    if constexpr (VEC % Wide<T>::n == 0) {
#pragma unroll
        for (int i = 0; i < VEC / Wide<T>::n; ++i) {
            const typename Wide<T>::type w = reinterpret_cast<const typename Wide<T>::type*>(at)[i];
#pragma unroll
            for (int j = 0; j < Wide<T>::n; ++j)
                p.v[i * Wide<T>::n + j] = w[j];
        }
    } else {
#pragma unroll
        for (int i = 0; i < VEC; ++i)
            p.v[i] = at[i];
    }
}
template <typename T, int VEC>
__device__ __forceinline__ void store_pack(const Pack<T, VEC>& p, T* at) {
    if constexpr (VEC % Wide<T>::n == 0) {
#pragma unroll
        for (int i = 0; i < VEC / Wide<T>::n; ++i) {
            typename Wide<T>::type w;
#pragma unroll
            for (int j = 0; j < Wide<T>::n; ++j)
                w[j] = p.v[i * Wide<T>::n + j];
            reinterpret_cast<typename Wide<T>::type*>(at)[i] = w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < VEC; ++i)
            at[i] = p.v[i];
    }
}

// Lane exchange by the vector unit's row operations (rows of 16 lanes): no LDS round trip.
template <int CTRL, int ROWS, typename V>
__device__ __forceinline__ V moved(V v) { // lanes without a source, and rows not in ROWS, get 0
    if constexpr (sizeof(V) == 4) {
        int i;
        __builtin_memcpy(&i, &v, 4);
        i = __builtin_amdgcn_update_dpp(0, i, CTRL, ROWS, 0xf, ROWS == 0xf);
        __builtin_memcpy(&v, &i, 4);
    } else {
        int i[2];
        __builtin_memcpy(i, &v, 8);
        i[0] = __builtin_amdgcn_update_dpp(0, i[0], CTRL, ROWS, 0xf, ROWS == 0xf);
        i[1] = __builtin_amdgcn_update_dpp(0, i[1], CTRL, ROWS, 0xf, ROWS == 0xf);
        __builtin_memcpy(&v, i, 8);
    }
    return v;
}
template <typename V>
__device__ __forceinline__ V of_lane(V v, int lane) { // lane: the same for the wavefront
    if constexpr (sizeof(V) == 4) {
        int i;
        __builtin_memcpy(&i, &v, 4);
        i = __builtin_amdgcn_readlane(i, lane);
        __builtin_memcpy(&v, &i, 4);
    } else {
        int i[2];
        __builtin_memcpy(i, &v, 8);
        i[0] = __builtin_amdgcn_readlane(i[0], lane);
        i[1] = __builtin_amdgcn_readlane(i[1], lane);
        __builtin_memcpy(&v, i, 8);
    }
    return v;
}
// Tokens of sequence b that count: lengths[b] held to [0, length], or all of them.
__device__ __forceinline__ int64_t tokens_of(const int32_t* lengths, int64_t b, int64_t length) {
    if (!lengths)
        return length;
    const int64_t n = lengths[b];
    return n < 0 ? 0 : n < length ? n : length;
}

// 2^f for |f| <= 1/2 and a little more: the interpolation of 2^f at the Chebyshev nodes of [-1/2, 1/2] by a polynomial
// (2^-55 off at most, its rounded coefficients included). The library's exponential spends a third of its
// instructions on its range.
__device__ __forceinline__ double exp2_part(double f) {
    double p = 4.4558179083360645e-10;
    p = fma(p, f, 7.074194297288521e-09);
    p = fma(p, f, 1.0178057087733941e-07);
    p = fma(p, f, 1.3215432535912375e-06);
    p = fma(p, f, 1.5252733841556773e-05);
    p = fma(p, f, 0.00015403530463724353);
    p = fma(p, f, 0.001333355814640647);
    p = fma(p, f, 0.009618129107587256);
    p = fma(p, f, 0.055504108664821625);
    p = fma(p, f, 0.24022650695910158);
    p = fma(p, f, 0.6931471805599453);
    return fma(p, f, 1.0);
}
// e^-|x| to 0.75 ulp: 2^(t - k) 2^k for t = -|x| log2(e), k the integer nearest to it. t - k is formed from the
// exact product with log2(e) in two parts: the rounded t alone would be off by |x| half steps (x = -20: 14 measured,
// 1.5 so). 0 for NaN.
__device__ __forceinline__ double exp_of_minus(double x) {
    const double a = fmin(fabs(x), 2000.0), k = rint(a * -1.4426950408889634);
    const double f = fma(a, -2.0355273740931033e-17, fma(a, -1.4426950408889634, -k));
    return __builtin_amdgcn_ldexp(exp2_part(f), (int)k);
}

// x * sigmoid(x). In 32 bits e^-x is the hardware's 2^t for the rounded t = -x log2(e), with what the rounding left,
// r = -x - t log(2), put in; without it the result is off by |x| half steps (18 on [-20, -10]). t is held to what 2^t can
// be: r makes up for it where x is below -87, until the reciprocal is 0 (results of 2^-119 and less; it has no
// denormals). The maximum is for 0 times infinity, at x = infinity.
__device__ __forceinline__ float silu(float x) {
    const float t = __builtin_amdgcn_fmed3f(x * -1.44269504088896341f, -150.0f, 126.0f);
    const float e = __builtin_amdgcn_exp2f(t), r = fmaf(t, -0.693147180559945309f, -x);
    return x * __builtin_amdgcn_rcpf(fmaxf(1.0f + fmaf(e, r, e), 1.0f));
}
__device__ __forceinline__ double silu(double x) {
    const double e = exp_of_minus(x);
    return x * ((x < 0.0 ? e : 1.0) / (1.0 + e));
}

} // namespace cnh
