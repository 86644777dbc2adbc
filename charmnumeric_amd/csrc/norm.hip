// Root-mean-square norm over the rows of a matrix, with the residual's addition in the same pass:
//   r = x + residual,  y = r / sqrt(mean(r^2) + eps) * weight
// The array path has no row reduction of its own (upstream reduces 1-D arrays only,
// src/executor_reduce.cpp:9-12), so this is one kernel of its own kind rather than a generated group.
//
// Bound by memory: x and residual are read once, r and y written once, five operations an element. A
// row stays in registers between the sum and the scaling, so nothing is read twice; rows of up to 64 x
// WAVES x VEC x ITEMS elements take this form, longer ones are swept a second time through the caches.
// Sums are kept in the element type (32 or 64 bits): per lane, then a tree over the wavefront, then one
// over the wavefronts of the row, always in the same order.
//
// A row gets one wavefront up to four packs a lane (1024 fp32 columns in 16-byte packs), four wavefronts up
// to eight packs a lane, sixteen beyond: one wavefront for 2048 columns took 110 us where four take
// 95.5 (16384 rows with a residual: 537 MB, 5.6 TB/s). 4 rows of 1024: 3.5 us, of which the launch and the
// fetching of the code are most. 777 odd rows of 1537 fp64: 8.2 us, 19 MB at 2.3 TB/s in accesses of one element.
#include "sequence.h"

#include <algorithm>
#include <limits>

using namespace cnh;

namespace {

template <typename T>
struct NormParams {
    int64_t rows, cols;
    const T* x;
    int64_t x_stride;
    const T* residual;
    int64_t residual_stride;
    T* residual_out;
    int64_t residual_out_stride;
    const T* weight;
    T eps;
    T* y;
    int64_t y_stride;
};

template <typename T>
__device__ __forceinline__ T wave_sum(T v) {
    v += moved<0xB1, 0xf>(v);  // quad_perm [1,0,3,2]
    v += moved<0x4E, 0xf>(v);  // quad_perm [2,3,0,1]
    v += moved<0x141, 0xf>(v); // row_half_mirror
    v += moved<0x140, 0xf>(v); // row_mirror
    return (of_lane(v, 0) + of_lane(v, 16)) + (of_lane(v, 32) + of_lane(v, 48));
}

// Sum over the WAVES wavefronts of a row, the same value in every lane.
template <typename T, int WAVES>
__device__ __forceinline__ T row_sum(T v, T* slots) {
    v = wave_sum(v);
    if constexpr (WAVES > 1) {
        if ((threadIdx.x & 63) == 0)
            slots[threadIdx.x >> 6] = v;
        __syncthreads();
        v = slots[0];
#pragma unroll
        for (int w = 1; w < WAVES; ++w)
            v += slots[w];
    }
    return v;
}

// ITEMS packs of VEC elements per lane hold the row (ITEMS 0: any length, two sweeps).
template <typename T, int VEC, int WAVES, int ITEMS>
__global__ __launch_bounds__(WAVES == 1 ? 256 : 64 * WAVES) void rms_norm_kernel(NormParams<T> p) {
    constexpr int LANES = 64 * WAVES, ROWS = WAVES == 1 ? 4 : 1;
    __shared__ T slots[WAVES];
    const int lane = WAVES == 1 ? (int)(threadIdx.x & 63) : (int)threadIdx.x;
    // With WAVES > 1 all lanes of a workgroup have the same rows, so the barriers below are met by all.
    for (int64_t row = (int64_t)blockIdx.x * ROWS + (WAVES == 1 ? (int)(threadIdx.x >> 6) : 0); row < p.rows;
         row += (int64_t)gridDim.x * ROWS) {
        const T* x = p.x + row * p.x_stride;
        const T* res = p.residual ? p.residual + row * p.residual_stride : nullptr;
        T* out = p.residual_out ? p.residual_out + row * p.residual_out_stride : nullptr;
        T* y = p.y + row * p.y_stride;
        T sum = 0;
        if constexpr (ITEMS > 0) {
            Pack<T, VEC> r[ITEMS];
#pragma unroll
            for (int i = 0; i < ITEMS; ++i) {
                const int64_t c = (int64_t)(i * LANES + lane) * VEC;
                if (c < p.cols)
                    load_pack(r[i], x + c);
            }
            if (res) {
                Pack<T, VEC> q[ITEMS];
#pragma unroll
                for (int i = 0; i < ITEMS; ++i) {
                    const int64_t c = (int64_t)(i * LANES + lane) * VEC;
                    if (c < p.cols)
                        load_pack(q[i], res + c);
                }
#pragma unroll
                for (int i = 0; i < ITEMS; ++i)
#pragma unroll
                    for (int j = 0; j < VEC; ++j)
                        r[i].v[j] += q[i].v[j];
            }
#pragma unroll
            for (int i = 0; i < ITEMS; ++i) {
                const int64_t c = (int64_t)(i * LANES + lane) * VEC;
                if (c < p.cols) {
                    if (out)
                        store_pack(r[i], out + c);
#pragma unroll
                    for (int j = 0; j < VEC; ++j)
                        sum += r[i].v[j] * r[i].v[j];
                }
            }
            sum = row_sum<T, WAVES>(sum, slots);
            const T scale = T(1) / sqrt(sum / (T)p.cols + p.eps);
#pragma unroll
            for (int i = 0; i < ITEMS; ++i) {
                const int64_t c = (int64_t)(i * LANES + lane) * VEC;
                if (c < p.cols) {
                    if (p.weight) {
                        Pack<T, VEC> w;
                        load_pack(w, p.weight + c);
#pragma unroll
                        for (int j = 0; j < VEC; ++j)
                            r[i].v[j] = r[i].v[j] * scale * w.v[j];
                    } else {
#pragma unroll
                        for (int j = 0; j < VEC; ++j)
                            r[i].v[j] *= scale;
                    }
                    store_pack(r[i], y + c);
                }
            }
        } else {
            for (int64_t c = (int64_t)lane * VEC; c < p.cols; c += LANES * VEC) {
                Pack<T, VEC> r;
                load_pack(r, x + c);
                if (res) {
                    Pack<T, VEC> q;
                    load_pack(q, res + c);
#pragma unroll
                    for (int j = 0; j < VEC; ++j)
                        r.v[j] += q.v[j];
                }
                // r waits in y for the second sweep: residual_out may be absent, and may be the residual
                if (out)
                    store_pack(r, out + c);
                store_pack(r, y + c);
#pragma unroll
                for (int j = 0; j < VEC; ++j)
                    sum += r.v[j] * r.v[j];
            }
            sum = row_sum<T, WAVES>(sum, slots);
            const T scale = T(1) / sqrt(sum / (T)p.cols + p.eps);
            // every lane reads back what it stored itself
            for (int64_t c = (int64_t)lane * VEC; c < p.cols; c += LANES * VEC) {
                Pack<T, VEC> r;
                load_pack(r, y + c);
                if (p.weight) {
                    Pack<T, VEC> w;
                    load_pack(w, p.weight + c);
#pragma unroll
                    for (int j = 0; j < VEC; ++j)
                        r.v[j] = r.v[j] * scale * w.v[j];
                } else {
#pragma unroll
                    for (int j = 0; j < VEC; ++j)
                        r.v[j] *= scale;
                }
                store_pack(r, y + c);
            }
        }
        if constexpr (WAVES > 1)
            __syncthreads(); // slots are written again for the next row
    }
}

template <typename T, int VEC, int WAVES, int ITEMS>
int launch(const NormParams<T>& p, hipStream_t st) {
    constexpr int ROWS = WAVES == 1 ? 4 : 1;
    // a launch takes fewer than 2^32 lanes: beyond a million workgroups each takes several rows
    const int64_t groups = std::min<int64_t>((p.rows + ROWS - 1) / ROWS, 1 << 20);
    rms_norm_kernel<T, VEC, WAVES, ITEMS><<<dim3((unsigned)groups), dim3(WAVES == 1 ? 256 : 64 * WAVES), 0, st>>>(p);
    CNH_HIP(hipGetLastError());
    return 0;
}

template <typename T, int VEC, int WAVES>
int launch_items(const NormParams<T>& p, hipStream_t st) {
    const int64_t per = 64 * WAVES * VEC;
    if (p.cols <= per)
        return launch<T, VEC, WAVES, 1>(p, st);
    if (p.cols <= 2 * per)
        return launch<T, VEC, WAVES, 2>(p, st);
    if (p.cols <= 4 * per)
        return launch<T, VEC, WAVES, 4>(p, st);
    if (p.cols <= 8 * per)
        return launch<T, VEC, WAVES, 8>(p, st);
    return launch<T, VEC, WAVES, 0>(p, st);
}

template <typename T, int VEC>
int launch_waves(const NormParams<T>& p, hipStream_t st) {
    if (p.cols <= 64 * VEC * 4)
        return launch_items<T, VEC, 1>(p, st);
    if (p.cols <= 256 * VEC * 8)
        return launch_items<T, VEC, 4>(p, st);
    return launch_items<T, VEC, 16>(p, st);
}

template <typename T>
int run(const cnh_rms_norm_args* a, hipStream_t st) {
    NormParams<T> p;
    p.rows = a->rows;
    p.cols = a->cols;
    p.x = static_cast<const T*>(a->x);
    p.x_stride = a->x_stride;
    p.residual = static_cast<const T*>(a->residual);
    p.residual_stride = a->residual_stride;
    p.residual_out = static_cast<T*>(a->residual_out);
    p.residual_out_stride = a->residual_out_stride;
    p.weight = static_cast<const T*>(a->weight);
    // an eps below the type's smallest number counts as that: it keeps a row of zeros one
    p.eps = a->eps > 0 ? std::max((T)a->eps, std::numeric_limits<T>::denorm_min()) : T(0);
    p.y = static_cast<T*>(a->y);
    p.y_stride = a->y_stride;
    constexpr int W = Wide<T>::n;
    const bool one = p.rows == 1;
    auto fits = [&](const void* ptr, int64_t stride) {
        return !ptr || (aligned_to(ptr, 16) && (one || stride % W == 0));
    };
    if (p.cols % W == 0 && fits(p.x, p.x_stride) && fits(p.residual, p.residual_stride) &&
        fits(p.residual_out, p.residual_out_stride) && fits(p.weight, 0) && fits(p.y, p.y_stride))
        return launch_waves<T, W>(p, st);
    return launch_waves<T, 1>(p, st);
}

} // namespace

extern "C" int cnh_rms_norm(const cnh_rms_norm_args* a, cnh_stream s) {
    CNH_CHECK(a != nullptr, -2, "cnh_rms_norm: null arguments");
    if (int rc = check_float_type(a->dtype, "cnh_rms_norm"))
        return rc;
    CNH_CHECK(a->rows >= 0 && a->cols >= 0, -2, "cnh_rms_norm: %lld rows of %lld columns", (long long)a->rows,
              (long long)a->cols);
    if (a->rows == 0 || a->cols == 0)
        return 0;
    CNH_CHECK(a->rows < ((int64_t)1 << 31) && a->cols < ((int64_t)1 << 31), -3,
              "cnh_rms_norm: %lld rows of %lld columns; both are below 2^31", (long long)a->rows, (long long)a->cols);
    CNH_CHECK(a->x && a->y, -2, "cnh_rms_norm: null x or y");
    CNH_CHECK(a->eps >= 0, -2, "cnh_rms_norm: eps %g is negative or no number", a->eps);
    CNH_CHECK(a->residual || !a->residual_out, -2, "cnh_rms_norm: residual_out without a residual");
    const int esz = dtype_size(a->dtype);
    auto extent = [&](const char* what, const void* ptr, int64_t stride) {
        return Extent{what, ptr, span_of(1, 0, a->rows, stride, a->cols) * esz};
    };
    const Extent y = extent("y", a->y, a->y_stride), out = extent("residual_out", a->residual_out, a->residual_out_stride),
                 x = extent("x", a->x, a->x_stride), res = extent("residual", a->residual, a->residual_stride),
                 w{"weight", a->weight, a->cols * esz};
    for (const Extent* e : {&y, &out, &x, &res, &w})
        if (int rc = check_extent(*e, esz, "cnh_rms_norm"))
            return rc;
    CNH_CHECK(rows_apart(1, 0, a->rows, a->y_stride, a->cols) &&
                  (!out.ptr || rows_apart(1, 0, a->rows, a->residual_out_stride, a->cols)),
              -2, "cnh_rms_norm: rows of an output overlap");
    for (const Extent* e : {&out, &x, &res, &w})
        CNH_CHECK(!overlap(y, *e), -2, "cnh_rms_norm: y overlaps %s", e->what);
    CNH_CHECK(!overlap(out, x) && !overlap(out, w), -2, "cnh_rms_norm: residual_out overlaps x or weight");
    CNH_CHECK(!overlap(out, res) || (out.ptr == res.ptr && (a->rows == 1 || a->residual_stride == a->residual_out_stride)),
              -2, "cnh_rms_norm: residual_out overlaps residual without being the same rows");
    if (int rc = ensure_init())
        return rc;
    DeviceScope dev;
    if (int rc = dev.enter())
        return rc;
    return a->dtype == CNH_F32 ? run<float>(a, as_stream(s)) : run<double>(a, as_stream(s));
}
