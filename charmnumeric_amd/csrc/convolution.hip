// Short causal convolution of every channel along its tokens (the depthwise filter in front of a
// state space scan), with the rows a sequence carries from one call to the next:
//   y[t] = act(bias + sum_k weight[k] * x[t - (taps - 1) + k]),   t < length,
// where x[-(taps - 1)] .. x[-1] are the rows of the state (zeros without one), and the state afterwards
// holds the last taps - 1 rows of the sequence. One token per sequence is the same call with length 1.
//
// Bound by memory: x is read once and y written once, 2 taps + 4 operations an element. Channels lie
// next to each other, so a lane owns 16 bytes of channels and a run of TOKENS rows, all of them loaded
// before the first is used; the taps - 1 rows before its first one are read a second time by the wavefront
// before it, mostly from the caches (3 in 11 rows for 4 taps). The runs cut a long prompt too, so that it
// fills the device. Short calls are bound by the launch and by fetching the code: hence few branches.
// 4 x 2048 x 4096 in fp32, 4 taps, silu: 45 us, 6.0 TB/s of x and y. One token of 64 x 4096: 4.1 us.
#include "sequence.h"

#include <algorithm>

using namespace cnh;

namespace {

template <typename T>
struct ConvParams {
    int64_t batch, length, channels;
    int64_t first_batch, first_run; // of this launch
    const T* x;
    int64_t x_batch_stride, x_stride;
    const T* weight;
    const T* bias;
    const T* state_in;
    T* state_out;
    const int32_t* lengths;
    T* y;
    int64_t y_batch_stride, y_stride;
};

// A workgroup is four wavefronts, each with 64 packs of channels and a run of tokens of its own, so rows are
// the same for a wavefront: their addresses and bounds are scalar work, and no branch stands between loads.
template <typename T, int VEC, int TAPS, int TOKENS, bool SILU>
__global__ __launch_bounds__(256) void convolution_kernel(ConvParams<T> p) {
    typedef Pack<T, VEC> Row;
    const uint32_t c = (blockIdx.x * 64 + threadIdx.x) * VEC; // channels are below 2^28
    if (c >= (uint32_t)p.channels)
        return;
    const int64_t run = p.first_run + blockIdx.y * 4 + __builtin_amdgcn_readfirstlane(threadIdx.y);
    const int64_t b = p.first_batch + blockIdx.z, t0 = run * TOKENS;
    if (t0 >= p.length && run > 0)
        return;
    const int64_t n = tokens_of(p.lengths, b, p.length);
    const T* x = p.x + b * p.x_batch_stride;
    const T* before = p.state_in ? p.state_in + b * (TAPS - 1) * p.channels : nullptr;
    // row t of the sequence with what came before it, t in [-(TAPS - 1), n); zeros elsewhere
    auto row = [&](int64_t t, Row& r) {
        const bool there = t >= 0 ? t < n : before != nullptr;
        const T* from = t >= 0 ? x + t * p.x_stride : before + (t + TAPS - 1) * p.channels;
        load_pack(r, (there ? from : p.weight) + c); // some row that exists
#pragma unroll
        for (int j = 0; j < VEC; ++j)
            r.v[j] = there ? r.v[j] : T(0);
    };
    Row w[TAPS], bias = {}, in[TAPS - 1 + TOKENS];
#pragma unroll
    for (int i = 0; i < TAPS - 1 + TOKENS; ++i)
        row(t0 - (TAPS - 1) + i, in[i]);
#pragma unroll
    for (int k = 0; k < TAPS; ++k)
        load_pack(w[k], p.weight + k * p.channels + c);
    if (p.bias)
        load_pack(bias, p.bias + c);
    // The wavefront with the first tokens is also the only reader of the state (a run is not shorter than
    // the state), so it may overwrite it in place: it has read what its own rows need, and reads all of
    // the last rows before it writes one.
    if (TAPS > 1 && run == 0 && p.state_out) {
        Row last[TAPS > 1 ? TAPS - 1 : 1];
#pragma unroll
        for (int j = 0; j < TAPS - 1; ++j)
            row(n - (TAPS - 1) + j, last[j]);
        T* after = p.state_out + b * (TAPS - 1) * p.channels + c;
#pragma unroll
        for (int j = 0; j < TAPS - 1; ++j)
            store_pack(last[j], after + j * p.channels);
    }
    T* y = p.y + b * p.y_batch_stride + t0 * p.y_stride;
#pragma unroll
    for (int i = 0; i < TOKENS; ++i) {
        const int64_t t = t0 + i;
        if (t >= p.length)
            break;
        Row out = bias;
#pragma unroll
        for (int k = 0; k < TAPS; ++k)
#pragma unroll
            for (int j = 0; j < VEC; ++j)
                out.v[j] += w[k].v[j] * in[i + k].v[j];
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            if (SILU)
                out.v[j] = silu(out.v[j]);
            out.v[j] = t < n ? out.v[j] : T(0);
        }
        store_pack(out, y + c);
        y += p.y_stride;
    }
}

template <typename T, int VEC, int TAPS, int TOKENS>
int launch(ConvParams<T> p, bool act, hipStream_t st) {
    const int64_t packs = (p.channels + VEC - 1) / VEC, runs = std::max<int64_t>((p.length + TOKENS - 1) / TOKENS, 1);
    const dim3 block(64, (unsigned)std::min<int64_t>(4, runs));
    // a grid takes 65535 in y and in z
    for (p.first_batch = 0; p.first_batch < p.batch; p.first_batch += 65535)
        for (p.first_run = 0; p.first_run < runs; p.first_run += 4 * 65535) {
            const dim3 grid((unsigned)((packs + 63) / 64), (unsigned)std::min<int64_t>((runs - p.first_run + 3) / 4, 65535),
                            (unsigned)std::min<int64_t>(p.batch - p.first_batch, 65535));
            if (act)
                convolution_kernel<T, VEC, TAPS, TOKENS, true><<<grid, block, 0, st>>>(p);
            else
                convolution_kernel<T, VEC, TAPS, TOKENS, false><<<grid, block, 0, st>>>(p);
        }
    CNH_HIP(hipGetLastError());
    return 0;
}

template <typename T, int VEC, int TAPS>
int launch_tokens(const ConvParams<T>& p, bool act, hipStream_t st) {
    return p.length <= 1 ? launch<T, VEC, TAPS, 1>(p, act, st) : launch<T, VEC, TAPS, 8>(p, act, st);
}

template <typename T, int VEC>
int launch_taps(const ConvParams<T>& p, int taps, bool act, hipStream_t st) {
    switch (taps) {
    case 1: return launch_tokens<T, VEC, 1>(p, act, st);
    case 2: return launch_tokens<T, VEC, 2>(p, act, st);
    case 3: return launch_tokens<T, VEC, 3>(p, act, st);
    case 4: return launch_tokens<T, VEC, 4>(p, act, st);
    case 5: return launch_tokens<T, VEC, 5>(p, act, st);
    case 6: return launch_tokens<T, VEC, 6>(p, act, st);
    case 7: return launch_tokens<T, VEC, 7>(p, act, st);
    default: return launch_tokens<T, VEC, 8>(p, act, st);
    }
}

template <typename T>
int run(const cnh_short_convolution_args* a, hipStream_t st) {
    ConvParams<T> p;
    p.batch = a->batch;
    p.length = a->length;
    p.channels = a->channels;
    p.x = static_cast<const T*>(a->x);
    p.x_batch_stride = a->x_batch_stride;
    p.x_stride = a->x_stride;
    p.weight = static_cast<const T*>(a->weight);
    p.bias = static_cast<const T*>(a->bias);
    p.state_in = static_cast<const T*>(a->state_in);
    p.state_out = static_cast<T*>(a->state_out);
    p.lengths = a->lengths;
    p.y = static_cast<T*>(a->y);
    p.y_batch_stride = a->y_batch_stride;
    p.y_stride = a->y_stride;
    constexpr int W = Wide<T>::n;
    auto fits = [&](const void* ptr, int64_t outer, int64_t inner) {
        return !ptr || (aligned_to(ptr, 16) && (p.batch == 1 || outer % W == 0) && (p.length <= 1 || inner % W == 0));
    };
    // Up to 64 channels fit a wavefront one to a lane, and packs would leave most lanes idle: 61 x 1024 tokens of
    // 64 channels take 9.4 us in fp32 and 15.3 in fp64, 14.1 and 19.4 in packs. 62 x 1024 of 96 take 14.3 and
    // 24.4, 14.4 and 23.8 in packs, and wider rows are faster in packs.
    if (p.channels > 64 && p.channels % W == 0 && fits(p.x, p.x_batch_stride, p.x_stride) && fits(p.y, p.y_batch_stride, p.y_stride) &&
        fits(p.weight, 0, 0) && fits(p.bias, 0, 0) && fits(p.state_in, 0, 0) && fits(p.state_out, 0, 0))
        return launch_taps<T, W>(p, a->taps, a->activation != 0, st);
    return launch_taps<T, 1>(p, a->taps, a->activation != 0, st);
}

} // namespace

extern "C" int cnh_short_convolution(const cnh_short_convolution_args* a, cnh_stream s) {
    const char* call = "cnh_short_convolution";
    CNH_CHECK(a != nullptr, -2, "%s: null arguments", call);
    if (int rc = check_float_type(a->dtype, call))
        return rc;
    CNH_CHECK(a->batch >= 0 && a->length >= 0 && a->channels >= 0, -2, "%s: batch %lld, length %lld, channels %lld", call,
              (long long)a->batch, (long long)a->length, (long long)a->channels);
    CNH_CHECK(a->taps >= 1 && a->taps <= 8, -3, "%s: %d taps; 1 to 8 are supported", call, a->taps);
    CNH_CHECK(a->activation == 0 || a->activation == 1, -2, "%s: activation %d is neither 0 (none) nor 1 (silu)", call,
              a->activation);
    if (a->batch == 0 || a->channels == 0 || (a->length == 0 && !a->state_out))
        return 0;
    CNH_CHECK(a->batch < ((int64_t)1 << 31) && a->length < ((int64_t)1 << 31) && a->channels < ((int64_t)1 << 28), -3,
              "%s: batch %lld, length %lld (below 2^31), channels %lld (below 2^28)", call, (long long)a->batch,
              (long long)a->length, (long long)a->channels);
    CNH_CHECK(a->weight && (a->length == 0 || (a->x && a->y)), -2, "%s: null x, weight or y", call);
    const int esz = dtype_size(a->dtype);
    const int64_t D = a->channels, state = a->batch * (a->taps - 1);
    auto rows = [&](int64_t n) {
        const __int128 b = (__int128)n * D * esz;
        return b < ((__int128)1 << 62) ? (int64_t)b : -1;
    };
    const Extent x{"x", a->x, span_of(a->batch, a->x_batch_stride, a->length, a->x_stride, D) * esz},
        y{"y", a->y, span_of(a->batch, a->y_batch_stride, a->length, a->y_stride, D) * esz},
        w{"weight", a->weight, rows(a->taps)}, bias{"bias", a->bias, rows(1)}, in{"state_in", a->state_in, rows(state)},
        out{"state_out", a->state_out, rows(state)}, len{"lengths", a->lengths, a->batch * 4};
    for (const Extent* e : {&x, &y, &w, &bias, &in, &out})
        if (int rc = check_extent(*e, esz, call))
            return rc;
    if (int rc = check_extent(len, 4, call))
        return rc;
    CNH_CHECK(rows_apart(a->batch, a->y_batch_stride, a->length, a->y_stride, D) || a->length == 0, -2,
              "%s: rows of y overlap", call);
    for (const Extent* e : {&x, &w, &bias, &in, &out, &len})
        CNH_CHECK(!overlap(y, *e), -2, "%s: y overlaps %s", call, e->what);
    for (const Extent* e : {&x, &w, &bias, &len})
        CNH_CHECK(!overlap(out, *e), -2, "%s: state_out overlaps %s", call, e->what);
    CNH_CHECK(!overlap(out, in) || out.ptr == in.ptr, -2, "%s: state_out overlaps state_in without being the same", call);
    if (int rc = ensure_init())
        return rc;
    DeviceScope dev;
    if (int rc = dev.enter())
        return rc;
    return a->dtype == CNH_F32 ? run<float>(a, as_stream(s)) : run<double>(a, as_stream(s));
}
