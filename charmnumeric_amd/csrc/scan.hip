// Selective state space scan: every channel of every sequence carries `states` numbers from token to
// token,
//   s_t = softplus(delta_t + delta_bias)                      (or delta_t + delta_bias as it is)
//   h_t[n] = exp(s_t A[n]) h_(t-1)[n] + s_t B_t[n] x_t,        n < states
//   y_t = (sum_n C_t[n] h_t[n] + skip x_t) z_t sigmoid(z_t)
// with A per channel and B, C shared by the channels of a token. One token per sequence is the same
// call with length 1.
//
// A lane owns NPL states of one channel in registers and walks the tokens; S neighbouring lanes share a
// channel with more states than that and add their parts of y over the lanes of a row. With S = 1 a
// wavefront is 64 neighbouring channels, x, delta, z and y move as whole lines, and B_t and C_t are the
// same for all lanes, so they come through the scalar cache and cost no vector register or LDS read.
//
// Per token and channel: 4 elements of memory and, per state, one exponential and five operations.
// A batch too small to fill the device is cut along the tokens: the recurrence is linear in h, so a
// piece of the sequence is summed up by the state it leaves when it starts from zero and by the sum of
// its steps (its decay is exp(A sum s)); a short pass over the pieces gives each its first state, and
// all pieces then run at once. That costs the exponentials twice, which is why it is left out as soon
// as half the vector units have a wavefront each (five eighths where B and C cannot be sent for ahead), and
// for prompts below 96 tokens.
//
// Prompts are bound by vector issue: a state of a token takes an exponential of 8.5 cycles and three to four
// operations of 4.3 to 5. One prompt of 8192 tokens, 2048 channels and 16 fp32 states, in 128 pieces: 60 us for
// what the pieces leave, 12 for their first states, 80 for the scan, vector issue busy 87 to 89 % of the time.
// Padded prompts leave it idle more (65 to 72 %): pieces are cut over the padded length, and those behind a
// sequence's end have nothing to do. One token of 128 x 4096 channels is bound by the states: 13.4 us, 75 MB at
// 5.6 TB/s.
#include "sequence.h"

#include <algorithm>
#include <limits>
#include <type_traits>

using namespace cnh;

namespace {

template <typename T>
struct ScanParams {
    int64_t batch, length, channels;
    int64_t first_batch; // of this launch
    int states, softplus;
    const T *x, *delta, *z;
    int64_t x_bs, delta_bs, z_bs; // elements between sequences
    uint32_t x_s, delta_s, z_s;   // bytes between tokens: half the scalar registers of a 64-bit stride
    const T* A;
    const T *B, *C;
    int64_t B_bs, C_bs;
    uint32_t B_s, C_s;
    const T *skip, *delta_bias;
    const T* state_in;
    T* state_out;
    const int32_t* lengths;
    T* y;
    int64_t y_bs;
    uint32_t y_s;
    int64_t piece;  // tokens per piece (a single token: sequences per workgroup)
    int pieces;     // 1: no cut
    T* carry;       // [batch][pieces][states][channels]: the state a piece leaves, then the one it starts from
    T* steps;       // [batch][pieces][channels]: sum of a piece's steps
};

// exp(s A) with what depends on A alone taken out of the loop. In 32 bits that is one multiplication and the
// hardware's base-2 exponential (1 ulp); the roundings of A log2(e) and of the product shift the result by |s A| half
// steps each, which the decay's own size makes harmless. An infinite rate is held to a finite one, so that no step
// (pieces behind a sequence's end) is no decay.
// In 64 bits the integer k nearest to t = s rate and the exact s rate - k leave the rounding of A log2(e) alone, |s A|
// half steps, about what rounding s A costs (110 measured at 100; the rounded t less k 188). Where t is beyond
// 2^52 the remainder is no small number any more: the polynomial's absolute value, finite as long as steps and
// rates are held to 1e22, keeps the result at 0 or infinity. The conversion of k saturates, and one instruction
// more holds the scaling to exponents that it takes (not to the lowest integer).
__device__ __forceinline__ float rate_of(float a) {
    return a != a ? a : fminf(fmaxf(a * 1.44269504088896341f, -3e38f), 3e38f);
}
__device__ __forceinline__ double held(double v) { return fmin(fmax(v, -1e22), 1e22); }
__device__ __forceinline__ double rate_of(double a) { return a != a ? a : held(a * 1.4426950408889634); }
__device__ __forceinline__ float decay(float s, float rate) { return __builtin_amdgcn_exp2f(s * rate); }
__device__ __forceinline__ double decay(double s, double rate) {
    const double v = held(s), k = rint(v * rate);
    int n; // the instruction itself: a C++ cast says nothing about what does not fit
    asm("v_cvt_i32_f64 %0, %1" : "=v"(n) : "v"(k));
    return __builtin_amdgcn_ldexp(fabs(exp2_part(fma(v, rate, -k))), max(min(n, 4096), -4096));
}

// The decay of many tokens, 2^f 2^k: it can leave the type's range where the state does not (states that grow from
// nothing or little, or large ones over a long piece). 2^f h scaled by 2^k leaves nothing at nothing, and the range
// only where the state itself is out of it. f is taken from the product before its rounding; exponents beyond `far`
// bring every number of the type out of its range.
template <typename T>
struct LongDecay {
    T part; // 2^f, |f| <= 1/2
    int k;
    __device__ __forceinline__ T operator()(T h) const { return ldexp(part * h, k); }
};
template <typename T>
__device__ __forceinline__ LongDecay<T> long_decay(T s, T rate) {
    constexpr T far = sizeof(T) == 4 ? T(600) : T(4400);
    const T t = s * rate, k = fmin(fmax(rint(t), -far), far);   // -far for no number, which f hands on
    const T f = fabs(t) > far ? T(0) : fma(s, rate, -k);
    if constexpr (sizeof(T) == 4)
        return {__builtin_amdgcn_exp2f(f), (int)k};
    else
        return {exp2_part(f), (int)k};
}

// log(1 + e^v). In 32 bits log(u) e / (u - 1) with u = 1 + e^v rounded (Kahan's log1p): the rounding of u cancels. e^v
// is the hardware's 2^t for the rounded t = v log2(e), with what the rounding left, v - t log(2), put in.
__device__ __forceinline__ float softplus(float v) {
    const float a = fmaxf(v, -200.0f), t = a * 1.44269504088896341f, e0 = __builtin_amdgcn_exp2f(t);
    const float e = fmaf(e0, fmaf(t, -0.693147180559945309f, a), e0), u = 1.0f + e, d = u - 1.0f;
    const float l = __builtin_amdgcn_logf(u) * 0.693147180559945309f;
    const float r = d == 0.0f ? e : l * (e * __builtin_amdgcn_rcpf(d));
    return v <= 20.0f ? r : v; // and what is no number
}
// In 64 bits max(v, 0) + log(1 + e) with e = e^-|v|, log(1 + e) = 2 atanh(e / (e + 2)) for small e and
// log 2 + 2 atanh((e - 1) / (e + 3)) above sqrt(2) - 1, so that the series' argument stays within 0.1716: ten
// terms leave 2^-58 of it.
__device__ __forceinline__ double softplus(double v) {
    const double e = exp_of_minus(v);
    const bool upper = e > 0.41421356237309503;
    const double num = upper ? e - 1.0 : e, den = e + (upper ? 3.0 : 2.0);
    double r = __builtin_amdgcn_rcp(den); // and Newton's steps
    r = fma(fma(-den, r, 1.0), r, r);
    r = fma(fma(-den, r, 1.0), r, r);
    double q = num * r;
    q = fma(fma(-den, q, num), r, q);
    const double z = q * q;
    double t = 1.0 / 21;
    t = fma(t, z, 1.0 / 19);
    t = fma(t, z, 1.0 / 17);
    t = fma(t, z, 1.0 / 15);
    t = fma(t, z, 1.0 / 13);
    t = fma(t, z, 1.0 / 11);
    t = fma(t, z, 1.0 / 9);
    t = fma(t, z, 1.0 / 7);
    t = fma(t, z, 1.0 / 5);
    t = fma(t, z, 1.0 / 3);
    const double l = fma(2.0 * q, z * t, 2.0 * q) + (upper ? 0.693147180559945309 : 0.0);
    return (v < 0.0 ? 0.0 : v) + l;
}

// Sum over S neighbouring lanes, in every one of them.
template <int S, typename T>
__device__ __forceinline__ T lanes_sum(T v) {
    if (S >= 2)
        v += moved<0xB1, 0xf>(v); // quad_perm [1,0,3,2]
    if (S >= 4)
        v += moved<0x4E, 0xf>(v); // quad_perm [2,3,0,1]
    if (S >= 8)
        v += moved<0x141, 0xf>(v); // row_half_mirror
    if (S >= 16)
        v += moved<0x140, 0xf>(v); // row_mirror
    return v;
}

// Element of a row that the wavefront shares, by the lane's byte offset (below 2^28): the row's address
// stays in scalar registers.
template <typename T>
__device__ __forceinline__ const T& at(const T* row, uint32_t bytes) {
    return *reinterpret_cast<const T*>(reinterpret_cast<const char*>(row) + bytes);
}
template <typename T>
__device__ __forceinline__ T& at(T* row, uint32_t bytes) {
    return *reinterpret_cast<T*>(reinterpret_cast<char*>(row) + bytes);
}

// v, or 0 (also for what is no number): by a mask in a lane's register, where scalar ones are scarce.
__device__ __forceinline__ float masked(float v, int32_t mask) { return __int_as_float(__float_as_int(v) & mask); }
__device__ __forceinline__ double masked(double v, int32_t mask) {
    return __hiloint2double(__double2hiint(v) & mask, __double2loint(v) & mask);
}

// v of lane U of every G neighbouring ones (G 2 or 4), in all of them.
template <int G, int U, typename T>
__device__ __forceinline__ T from_lane(T v) {
    return moved<(G == 4 ? U * 0x55 : U ? 0xF5 : 0xA0), 0xf>(v);
}

// A row so many bytes further.
template <typename T>
__device__ __forceinline__ const T* on(const T* row, int64_t bytes) {
    return reinterpret_cast<const T*>(reinterpret_cast<const char*>(row) + bytes);
}
template <typename T>
__device__ __forceinline__ T* on(T* row, int64_t bytes) {
    return reinterpret_cast<T*>(reinterpret_cast<char*>(row) + bytes);
}

// Memory that no kernel in flight writes, for loads at addresses the whole wavefront shares.
template <typename T>
using Uniform = const __attribute__((address_space(4))) T;

// A row of B or C in scalar registers: BYTES of them, from an address aligned to 4.
template <int BYTES>
struct ScalarRow;
template <>
struct ScalarRow<16> {
    typedef uint32_t type __attribute__((ext_vector_type(4), aligned(4)));
};
template <>
struct ScalarRow<32> {
    typedef uint32_t type __attribute__((ext_vector_type(8), aligned(4)));
};
template <>
struct ScalarRow<64> {
    typedef uint32_t type __attribute__((ext_vector_type(16), aligned(4)));
};

// The states of a lane: NPL one behind the other from n0 on when FULL (all of them exist, the rows of A and of
// the states are aligned for wide accesses and, with S > 1, those of B and C too); every S-th from n0 on
// otherwise, so that the lanes of a channel read neighbouring elements.
template <int S, bool FULL>
constexpr int STEP = FULL ? 1 : S;
template <int NPL, int S, bool FULL>
__device__ __forceinline__ int first_state(uint32_t lane) {
    return (int)(lane % S) * (FULL ? NPL : 1);
}

// Is the lane's i-th state one of the channel's? plan_of() gives a channel more than half of the states that its
// lanes could hold (one lane of four holds one to four), so only the second half of a lane's can be missing. Those
// are worked on with the last state's B and C, and kept out of every sum and store whatever becomes of them: a
// select less than zeros in their place, and an infinite step times input stays out of y.
template <int NPL, int S, bool FULL>
__device__ __forceinline__ bool there(int i, int n0, int states) {
    return FULL || i < (NPL == 4 && S == 1 ? 1 : NPL / 2) || n0 + i * STEP<S, FULL> < states;
}

// Those of one token's B or C.
template <typename T, int NPL, int S, bool FULL>
__device__ __forceinline__ void load_states(T (&v)[NPL], const T* row, int n0, int states) {
    if constexpr (S == 1) {
        Uniform<T>* u = (Uniform<T>*)(uintptr_t)row;
#pragma unroll
        for (int i = 0; i < NPL; ++i)
            v[i] = u[there<NPL, S, FULL>(i, 0, states) ? i : states - 1];
    } else if constexpr (FULL) {
        Pack<T, NPL> q;
        load_pack(q, row + n0);
#pragma unroll
        for (int i = 0; i < NPL; ++i)
            v[i] = q.v[i];
    } else {
        // no branches between the loads
#pragma unroll
        for (int i = 0; i < NPL; ++i)
            v[i] = row[there<NPL, S, FULL>(i, n0, states) ? n0 + i * STEP<S, FULL> : states - 1];
    }
}

// Those of a lane's own channel, from a row of `states` elements.
template <typename T, int NPL, int S, bool FULL>
__device__ __forceinline__ void own_states(Pack<T, NPL>& v, const T* row, int n0, int states) {
    if constexpr (FULL) {
        load_pack(v, row + n0);
    } else {
#pragma unroll
        for (int i = 0; i < NPL; ++i)
            v.v[i] = n0 + i * STEP<S, FULL> < states ? row[n0 + i * STEP<S, FULL>] : T(0);
    }
}

template <typename T, int NPL, int S, bool FULL>
__device__ __forceinline__ void store_states(const Pack<T, NPL>& v, T* row, int n0, int states) {
    if constexpr (FULL) {
        store_pack(v, row + n0);
    } else {
#pragma unroll
        for (int i = 0; i < NPL; ++i)
            if (n0 + i * STEP<S, FULL> < states)
                row[n0 + i * STEP<S, FULL>] = v.v[i];
    }
}

// PARTIAL: what a piece leaves when it starts from zero; otherwise the scan itself.
template <typename T, int NPL, int S, bool FULL, bool PARTIAL>
__global__ __launch_bounds__(64) void scan_kernel(ScanParams<T> p) {
    // Tokens whose x, delta and z are on their way while others are worked on. With S > 1 their rows of B and
    // C are loaded together: no more than 64 registers of them.
    constexpr int AHEAD = S > 1 ? std::min(4, 128 / (NPL * (int)sizeof(T))) : 4;
    const uint32_t lane = blockIdx.x * 64 + threadIdx.x; // below 2^28: 16 lanes for each of 2^24 channels
    const uint32_t d_own = lane / S;
    const bool live = d_own < (uint32_t)p.channels;
    // lanes past the last channel work on the last one and store nothing: the wavefront stays whole
    const uint32_t d = live ? d_own : (uint32_t)p.channels - 1;
    const int n0 = first_state<NPL, S, FULL>(lane);
    const uint32_t off = d * (uint32_t)sizeof(T);
    const bool first = n0 == 0;
    const int64_t piece = blockIdx.y;
    Pack<T, NPL> rate;
    own_states<T, NPL, S, FULL>(rate, p.A + (int64_t)d * p.states, n0, p.states);
#pragma unroll
    for (int i = 0; i < NPL; ++i)
        rate.v[i] = rate_of(rate.v[i]);
    const T bias = p.delta_bias ? p.delta_bias[d] : T(0), skip = p.skip ? p.skip[d] : T(0);
    int32_t keep = p.skip ? -1 : 0; // without a skip nothing of x is added, infinities neither
    asm("" : "+v"(keep));

    const int64_t b = p.first_batch + blockIdx.z;
    const int64_t n = tokens_of(p.lengths, b, p.length);
    const int64_t begin = piece * p.piece, stop = std::min(begin + p.piece, p.length), end = std::min(stop, n);
    // rows: the same for the whole wavefront; a lane adds its channel
    const T* xp = p.x + b * p.x_bs;
    const T* dp = p.delta + b * p.delta_bs;
    const T* zp = p.z ? p.z + b * p.z_bs : nullptr;
    // without a gate the loads of z repeat those of x: cheaper than a branch around each
    const T* zq = zp ? zp : xp;
    const uint32_t zq_s = zp ? p.z_s : p.x_s;
    T* yp = p.y + b * p.y_bs;
    T* slot = p.carry + ((b * p.pieces + piece) * p.states + n0) * p.channels + d;
    Pack<T, NPL> h = {};
    if (!PARTIAL) {
        if (p.pieces > 1) {
#pragma unroll
            for (int i = 0; i < NPL; ++i)
                h.v[i] = FULL || n0 + i * STEP<S, FULL> < p.states ? slot[(int64_t)(i * STEP<S, FULL>) * p.channels] : T(0);
        } else if (p.state_in) {
            own_states<T, NPL, S, FULL>(h, p.state_in + (b * p.channels + d) * p.states, n0, p.states);
        }
    }
    T steps = 0;
    // M tokens from t0 on; their steps and gates first, so that the branches on what the call has come once
    const T *Bt_row = on(p.B + b * p.B_bs, begin * (int64_t)p.B_s),
            *Ct_row = on(p.C + b * p.C_bs, begin * (int64_t)p.C_s);
    T* y_row = on(yp, begin * (int64_t)p.y_s);
    // B and C one token ahead in scalar registers, where two tokens' rows of both fit them.
    constexpr bool EARLY = S == 1 && FULL && NPL * sizeof(T) <= 64;
    typedef typename ScalarRow<EARLY ? NPL * sizeof(T) : 16>::type Scalars;
    Scalars B_early = {}, C_early = {};
    int left = end > begin ? (int)(end - begin) : 0; // rows not sent for yet
    auto send = [&]() { // behind the last row that one again
        B_early = *(Uniform<Scalars>*)(uintptr_t)Bt_row;
        if constexpr (!PARTIAL)
            C_early = *(Uniform<Scalars>*)(uintptr_t)Ct_row;
        --left;
        Bt_row = on(Bt_row, left > 0 ? p.B_s : 0);
        Ct_row = on(Ct_row, left > 0 ? p.C_s : 0);
    };
    if constexpr (EARLY)
        if (left > 0)
            send();
    auto tokens = [&](auto count, const T* xc, const T* dc, const T* zc) {
        constexpr int M = decltype(count)::value;
        // With S > 1 B and C are vector loads: all of the group's before the first is waited for. (Scalar
        // registers have no room for that.)
        T Bt[S > 1 ? M : 1][NPL], Ct[S > 1 && !PARTIAL ? M : 1][NPL];
        if constexpr (S > 1) {
#pragma unroll
            for (int u = 0; u < M; ++u) {
                load_states<T, NPL, S, FULL>(Bt[u], on(Bt_row, u * (int64_t)p.B_s), n0, p.states);
                if constexpr (!PARTIAL)
                    load_states<T, NPL, S, FULL>(Ct[u], on(Ct_row, u * (int64_t)p.C_s), n0, p.states);
            }
        }
        T s[M], gate[M];
        // The lanes of a channel have its tokens in common: each of G neighbours works out the steps and
        // gates of M / G tokens and hands them to the others.
        constexpr int G = M % 4 == 0 && S >= 4 ? 4 : M % 2 == 0 && S >= 2 ? 2 : 1;
        const int turn = (int)(lane % G);
        auto shared = [&](const T* in, T* out, auto f) {
            if constexpr (G == 1) {
#pragma unroll
                for (int u = 0; u < M; ++u)
                    out[u] = f(in[u]);
            } else {
#pragma unroll
                for (int u = 0; u < M; u += G) {
                    T mine = in[u];
#pragma unroll
                    for (int i = 1; i < G; ++i) {
                        const T other = in[u + i];
                        mine = turn == i ? other : mine;
                    }
                    mine = f(mine);
                    out[u] = from_lane<G, 0>(mine);
                    out[u + 1] = from_lane<G, 1>(mine);
                    if constexpr (G == 4) {
                        out[u + 2] = from_lane<G, 2>(mine);
                        out[u + 3] = from_lane<G, 3>(mine);
                    }
                }
            }
        };
        if (p.softplus) {
            shared(dc, s, [&](T v) { return softplus(v + bias); });
        } else {
#pragma unroll
            for (int u = 0; u < M; ++u)
                s[u] = dc[u] + bias;
        }
        if (!PARTIAL && zp)
            shared(zc, gate, [&](T v) { return silu(v); });
#pragma unroll
        for (int u = 0; u < M; ++u) {
            const T sx = s[u] * xc[u];
            constexpr bool GROUPED = S > 1;
            T(&B)[NPL] = Bt[GROUPED ? u : 0];
            if constexpr (EARLY) {
                // These rows have been on their way since the last token. They are waited for here, the
                // next token's are sent for, and only then the work begins that covers their flight:
                // scalar loads return in any order, so a wait further down would wait for both.
                asm volatile("" : : "s"(B_early));
                if constexpr (!PARTIAL)
                    asm volatile("" : : "s"(C_early));
                __builtin_amdgcn_sched_barrier(0);
                const Scalars B_now = B_early, C_now = C_early;
                send();
                __builtin_amdgcn_sched_barrier(0);
                __builtin_memcpy(B, &B_now, sizeof B);
                if constexpr (!PARTIAL)
                    __builtin_memcpy(Ct[0], &C_now, sizeof Ct[0]);
            } else {
                if constexpr (!GROUPED)
                    load_states<T, NPL, S, FULL>(B, Bt_row, n0, p.states);
                Bt_row = on(Bt_row, p.B_s);
            }
            if constexpr (PARTIAL) {
                steps += s[u];
#pragma unroll
                for (int i = 0; i < NPL; ++i)
                    h.v[i] = decay(s[u], rate.v[i]) * h.v[i] + sx * B[i];
            } else {
                T(&C)[NPL] = Ct[GROUPED ? u : 0];
                if constexpr (!GROUPED && !EARLY)
                    load_states<T, NPL, S, FULL>(C, Ct_row, n0, p.states);
                if constexpr (!EARLY)
                    Ct_row = on(Ct_row, p.C_s);
                T sum = 0;
#pragma unroll
                for (int i = 0; i < NPL; ++i) {
                    h.v[i] = decay(s[u], rate.v[i]) * h.v[i] + sx * B[i];
                    sum += there<NPL, S, FULL>(i, n0, p.states) ? C[i] * h.v[i] : T(0);
                }
                sum = lanes_sum<S>(sum) + skip * masked(xc[u], keep);
                if (zp)
                    sum *= gate[u];
                if (first && live)
                    at(y_row, off) = sum;
                y_row = on(y_row, p.y_s);
            }
        }
    };
    // Whole groups of tokens, the next group's x, delta and z on their way meanwhile, then what is left.
    // Behind the last group its last token is fetched again: no branch stands between a load and its wait.
    const T *x_row = on(xp, begin * (int64_t)p.x_s), *d_row = on(dp, begin * (int64_t)p.delta_s),
            *z_row = on(zq, begin * (int64_t)zq_s);
    const int groups = end > begin ? (int)((end - begin) / AHEAD) : 0, rest = end > begin ? (int)((end - begin) % AHEAD) : 0;
    if (groups > 0) {
        T xs[AHEAD], ds[AHEAD], zs[AHEAD];
        auto fetch = [&](uint32_t x_on, uint32_t d_on, uint32_t z_on) {
#pragma unroll
            for (int u = 0; u < AHEAD; ++u) {
                xs[u] = at(x_row, off);
                ds[u] = at(d_row, off);
                zs[u] = PARTIAL ? T(0) : at(z_row, off);
                x_row = on(x_row, x_on);
                d_row = on(d_row, d_on);
                z_row = on(z_row, z_on);
            }
        };
        fetch(p.x_s, p.delta_s, zq_s);
        for (int g = 1; g <= groups; ++g) {
            T xc[AHEAD], dc[AHEAD], zc[AHEAD];
#pragma unroll
            for (int u = 0; u < AHEAD; ++u) {
                xc[u] = xs[u];
                dc[u] = ds[u];
                zc[u] = zs[u];
            }
            const bool more = g < groups;
            x_row = on(x_row, more ? 0 : -(int64_t)p.x_s);
            d_row = on(d_row, more ? 0 : -(int64_t)p.delta_s);
            z_row = on(z_row, more ? 0 : -(int64_t)zq_s);
            fetch(more ? p.x_s : 0, more ? p.delta_s : 0, more ? zq_s : 0);
            tokens(std::integral_constant<int, AHEAD>(), xc, dc, zc);
        }
        x_row = on(x_row, p.x_s);
        d_row = on(d_row, p.delta_s);
        z_row = on(z_row, zq_s);
    }
    for (int r = 0; r < rest; ++r) {
        const T xc = at(x_row, off), dc = at(d_row, off), zc = PARTIAL ? T(0) : at(z_row, off);
        x_row = on(x_row, p.x_s);
        d_row = on(d_row, p.delta_s);
        z_row = on(z_row, zq_s);
        tokens(std::integral_constant<int, 1>(), &xc, &dc, &zc);
    }
    if constexpr (PARTIAL) {
        if (live) {
#pragma unroll
            for (int i = 0; i < NPL; ++i)
                if (FULL || n0 + i * STEP<S, FULL> < p.states)
                    slot[(int64_t)(i * STEP<S, FULL>) * p.channels] = h.v[i];
            if (first)
                p.steps[(b * p.pieces + piece) * p.channels + d] = steps;
        }
    } else {
        if (first && live)
            for (int64_t t = std::max(begin, end); t < stop; ++t)
                at(on(yp, t * (int64_t)p.y_s), off) = T(0);
        if (p.state_out && piece == p.pieces - 1 && live) {
            store_states<T, NPL, S, FULL>(h, p.state_out + (b * p.channels + d) * p.states, n0, p.states);
        }
    }
}

// The state each piece starts from, in place of the one it leaves: 64 channels of one state per workgroup,
// up to kSegments x GROUP pieces a round (as many segments as the pieces need). A lane loads its GROUP
// pieces at once, folds them to one, takes what the segments before it leave from shared memory and walks
// its pieces again in registers. 128 pieces of 2048 x 16 fp32 states: 11.9 us (10.7 with decays that left the
// type's range; 22.5 then with one lane per channel that walks all pieces by itself and waits for memory once per
// GROUP of them).
constexpr int kSegments = 8, kGroup = 8;
template <typename T>
__global__ __launch_bounds__(64 * kSegments) void carry_kernel(ScanParams<T> p) {
    constexpr int GROUP = kGroup;
    __shared__ T left_by[kSegments][64];
    __shared__ LongDecay<T> decay_of[kSegments][64];
    const int seg = threadIdx.y, lane = threadIdx.x, segments = blockDim.y;
    const int64_t own = (int64_t)blockIdx.x * 64 + lane;
    const bool live = own < p.channels;
    const int64_t d = live ? own : p.channels - 1;
    const int n = blockIdx.y;
    const int64_t b = p.first_batch + blockIdx.z;
    const T rate = rate_of(p.A[d * p.states + n]);
    T start = p.state_in ? p.state_in[(b * p.channels + d) * p.states + n] : T(0); // of the round
    for (int c0 = 0; c0 < p.pieces; c0 += segments * GROUP) {
        const int c1 = c0 + seg * GROUP;
        T left[GROUP], steps[GROUP];
        LongDecay<T> decays[GROUP];
#pragma unroll
        for (int i = 0; i < GROUP; ++i) {
            const int64_t c = b * p.pieces + c1 + i;
            const bool in = c1 + i < p.pieces - 1; // nothing starts behind the last piece
            left[i] = in ? p.carry[(c * p.states + n) * p.channels + d] : T(0);
            steps[i] = in ? p.steps[c * p.channels + d] : T(0);
        }
        T h = 0, sum = 0;
#pragma unroll
        for (int i = 0; i < GROUP; ++i) {
            decays[i] = long_decay(steps[i], rate);
            h = decays[i](h) + left[i];
            sum += steps[i];
        }
        left_by[seg][lane] = h;
        decay_of[seg][lane] = long_decay(sum, rate);
        __syncthreads();
        T at = start;
        h = start;
        for (int s = 0; s < segments; ++s) {
            if (s == seg)
                h = at;
            at = decay_of[s][lane](at) + left_by[s][lane];
        }
        start = at;
#pragma unroll
        for (int i = 0; i < GROUP; ++i) {
            if (c1 + i < p.pieces && live)
                p.carry[((b * p.pieces + c1 + i) * p.states + n) * p.channels + d] = h;
            h = decays[i](h) + left[i];
        }
        __syncthreads(); // the next round writes the shared memory again
    }
}

// One token per sequence. The states are what moves: they are read and written once as 16-byte
// accesses, a lane keeps its channel's A through the sequences of its slice, and the next sequence's
// operands are on their way while the present one is worked on (128 x 4096 x 16 fp32 states: 13.4 us).
template <typename T, int NPL, int S, bool FULL>
__global__ __launch_bounds__(256) void token_kernel(ScanParams<T> p) {
    const uint32_t lane = blockIdx.x * 256 + threadIdx.x;
    const uint32_t d_own = lane / S;
    const bool live = d_own < (uint32_t)p.channels;
    const uint32_t d = live ? d_own : (uint32_t)p.channels - 1;
    const int n0 = first_state<NPL, S, FULL>(lane);
    const int64_t begin = blockIdx.y * p.piece, end = std::min(begin + p.piece, p.batch);
    Pack<T, NPL> rate;
    own_states<T, NPL, S, FULL>(rate, p.A + (int64_t)d * p.states, n0, p.states);
#pragma unroll
    for (int i = 0; i < NPL; ++i)
        rate.v[i] = rate_of(rate.v[i]);
    const T bias = p.delta_bias ? p.delta_bias[d] : T(0), skip = p.skip ? p.skip[d] : T(0);
    const int32_t keep = p.skip ? -1 : 0;
    struct Operands {
        T x, delta, z, B[NPL], C[NPL];
        Pack<T, NPL> h;
        bool there;
    };
    auto fetch = [&](int64_t b, Operands& o) {
        o.there = tokens_of(p.lengths, b, 1) > 0;
        o.x = (p.x + b * p.x_bs)[d];
        o.delta = (p.delta + b * p.delta_bs)[d];
        o.z = p.z ? (p.z + b * p.z_bs)[d] : T(0);
        load_states<T, NPL, S, FULL>(o.B, p.B + b * p.B_bs, n0, p.states);
        load_states<T, NPL, S, FULL>(o.C, p.C + b * p.C_bs, n0, p.states);
        o.h = Pack<T, NPL>{};
        if (p.state_in)
            own_states<T, NPL, S, FULL>(o.h, p.state_in + (b * p.channels + d) * p.states, n0, p.states);
    };
    Operands next;
    fetch(begin, next);
    for (int64_t b = begin; b < end; ++b) {
        Operands o = next;
        fetch(std::min(b + 1, end - 1), next);
        T out = 0;
        if (o.there) {
            T s = o.delta + bias;
            if (p.softplus)
                s = softplus(s);
            const T sx = s * o.x;
#pragma unroll
            for (int i = 0; i < NPL; ++i) {
                o.h.v[i] = decay(s, rate.v[i]) * o.h.v[i] + sx * o.B[i];
                out += there<NPL, S, FULL>(i, n0, p.states) ? o.C[i] * o.h.v[i] : T(0);
            }
            out = lanes_sum<S>(out) + skip * masked(o.x, keep);
            if (p.z)
                out *= silu(o.z);
        }
        if (live) {
            if (n0 == 0)
                (p.y + b * p.y_bs)[d] = out;
            if (p.state_out)
                store_states<T, NPL, S, FULL>(o.h, p.state_out + (b * p.channels + d) * p.states, n0, p.states);
        }
    }
}

// States per lane, lanes per channel and pieces of a call: host arithmetic on its sizes alone, so that
// the workspace it needs can be asked for without a device.
struct Plan {
    int npl, lanes;
    int64_t piece;
    int pieces;
    int64_t bytes;
};

constexpr int64_t kUnits = 256 * 4; // vector units of the device

Plan plan_of(const cnh_state_scan_args* a) {
    Plan q;
    const int64_t N = a->states, D = a->channels, L = a->length;
    auto lanes = [&](int npl) {
        int s = 1;
        while (npl * s < N)
            s *= 2;
        return s;
    };
    auto waves = [&](int s) { return a->batch * ((D * s + 63) / 64); };
    // Either way more than half of npl x lanes states exist, or one of four: there() builds on that.
    // Few states per lane spread a small call over more lanes and make a single token's states one
    // 16-byte access each; many states per lane share a token's step and gate. Few as long as the
    // pieces of 32 tokens that the call could be cut into would not fill the device with many.
    // For 33 to 64 states few are taken always (64 states, 2048 channels, sixteen a lane and four: 16 x 100
    // tokens 109 and 110 us in fp32, 384 and 300 in fp64; 4 x 300 tokens 133 and 103, 472 and 224; with 50 states
    // 16 x 100 tokens would take 88 instead of 122, 249 instead of 343).
    // Where a lane's many are not all there, few are faster in uncut calls with less than a wavefront per unit
    // (many and few, 22 x 200 tokens of 2048 channels, 12 states: 172 and 103 us in fp32, 344 and 302 in fp64; 23 x 100,
    // 20 states: 126 and 93, 319 and 269), many beyond (62 x 200 tokens, 10 states: 193 and 265, 471 and 734;
    // 65 x 100, 20 states: 204 and 264, 682 and 714; 130 x 50, 31 states: 206 and 275, 628 and 733).
    const int many = N <= 8 || (N > 64 && N <= 128) ? 8 : N <= 16 || N > 128 ? 16 : 32;
    const int64_t wm = waves(lanes(many));
    const bool sparse = N != many && wm > kUnits * 5 / 8 && wm < kUnits;
    q.npl = many;
    if (N <= 64 && (N > 32 || N <= 4 || L <= 1 || wm * std::max<int64_t>(1, L / 32) < 2 * kUnits || sparse))
        q.npl = 4;
    q.lanes = lanes(q.npl);
    q.pieces = 1;
    const int64_t w = waves(q.lanes);
    if (L <= 1) {
        // sequences per slice: eight wavefronts on each vector unit, or what there is
        const int64_t row = (D * q.lanes + 63) / 64, slices = std::max<int64_t>(1, std::min(a->batch, 8 * kUnits / std::max<int64_t>(row, 1)));
        q.piece = std::max<int64_t>(1, (a->batch + slices - 1) / slices);
        q.piece = std::max(q.piece, (a->batch + 65534) / 65535);
    } else {
        // Measured with 300 tokens of 2048 fp32 channels, 16 states: 16 sequences (512 wavefronts) 126 us
        // uncut, 101 us in 8 pieces; 24 sequences (768) 134 us uncut, 140 us in 3. With 256 channels of
        // 2 sequences: 64 tokens 17 us uncut, 23 us in 4 pieces; 128 tokens 31 and 23 us. Where B and C do
        // not travel ahead in scalar registers a lone wavefront waits for them: 17 sequences (544 wavefronts)
        // of 32 states 312 us uncut, 175 in 7 pieces; fp64 12 states 506 and 335.
        const bool early = q.lanes == 1 && N == q.npl && N * dtype_size(a->dtype) <= 64;
        if (w <= (early ? kUnits / 2 : kUnits * 5 / 8) && w > 0 && L >= 96)
            q.pieces = (int)std::min(4 * kUnits / w, L / 16);
        q.piece = (L + q.pieces - 1) / q.pieces;
        q.pieces = (int)((L + q.piece - 1) / q.piece);
    }
    q.bytes = q.pieces > 1 ? a->batch * q.pieces * (N + 1) * D * dtype_size(a->dtype) : 0;
    return q;
}

template <typename T, int NPL, int S, bool FULL>
int launch(ScanParams<T> p, hipStream_t st) {
    if constexpr (NPL == 4 || S == 16) // what single tokens take
        if (p.length == 1) {
            const dim3 grid((unsigned)((p.channels * S + 255) / 256), (unsigned)((p.batch + p.piece - 1) / p.piece));
            token_kernel<T, NPL, S, FULL><<<grid, 256, 0, st>>>(p);
            CNH_HIP(hipGetLastError());
            return 0;
        }
    // one wavefront per workgroup: few long-running wavefronts spread evenly over the device
    const unsigned gx = (unsigned)((p.channels * S + 63) / 64);
    for (p.first_batch = 0; p.first_batch < p.batch; p.first_batch += 65535) { // what a grid takes
        const unsigned gz = (unsigned)std::min<int64_t>(p.batch - p.first_batch, 65535);
        if (p.pieces > 1) {
            scan_kernel<T, NPL, S, FULL, true><<<dim3(gx, p.pieces - 1, gz), 64, 0, st>>>(p);
            const int segments = std::min(kSegments, (p.pieces + kGroup - 1) / kGroup);
            carry_kernel<T><<<dim3((unsigned)((p.channels + 63) / 64), p.states, gz), dim3(64, segments), 0, st>>>(p);
        }
        scan_kernel<T, NPL, S, FULL, false><<<dim3(gx, p.pieces, gz), 64, 0, st>>>(p);
    }
    CNH_HIP(hipGetLastError());
    return 0;
}

template <typename T, int NPL, int S>
int launch_full(const ScanParams<T>& p, bool wide, hipStream_t st) {
    const bool own = aligned_to(p.A, 16) && aligned_to(p.state_in, 16) && aligned_to(p.state_out, 16);
    if (p.states == NPL * S && own && (S == 1 || wide))
        return launch<T, NPL, S, true>(p, st);
    return launch<T, NPL, S, false>(p, st);
}

template <typename T>
int run(const cnh_state_scan_args* a, const Plan& q, hipStream_t st) {
    ScanParams<T> p;
    auto in = [](const void* v) { return static_cast<const T*>(v); };
    p.batch = a->batch;
    p.length = a->length;
    p.channels = a->channels;
    p.states = (int)a->states;
    p.softplus = a->softplus;
    auto bytes = [](int64_t stride) { return (uint32_t)(stride * (int64_t)sizeof(T)); }; // checked by the caller
    p.x = in(a->x), p.x_bs = a->x_batch_stride, p.x_s = bytes(a->x_stride);
    p.delta = in(a->delta), p.delta_bs = a->delta_batch_stride, p.delta_s = bytes(a->delta_stride);
    p.z = in(a->z), p.z_bs = a->z_batch_stride, p.z_s = bytes(a->z_stride);
    p.A = in(a->A);
    p.B = in(a->B), p.B_bs = a->B_batch_stride, p.B_s = bytes(a->B_stride);
    p.C = in(a->C), p.C_bs = a->C_batch_stride, p.C_s = bytes(a->C_stride);
    p.skip = in(a->skip);
    p.delta_bias = in(a->delta_bias);
    p.state_in = in(a->state_in);
    p.state_out = static_cast<T*>(a->state_out);
    p.lengths = a->lengths;
    p.y = static_cast<T*>(a->y), p.y_bs = a->y_batch_stride, p.y_s = bytes(a->y_stride);
    p.piece = q.piece;
    p.pieces = q.pieces;
    p.carry = static_cast<T*>(a->workspace);
    p.steps = p.carry ? p.carry + p.batch * p.pieces * p.states * p.channels : nullptr;
    constexpr int W = Wide<T>::n;
    auto fits = [&](const void* ptr, int64_t outer, int64_t inner) {
        return aligned_to(ptr, 16) && (p.batch == 1 || outer % W == 0) && (p.length <= 1 || inner % W == 0);
    };
    const bool wide = fits(p.B, p.B_bs, a->B_stride) && fits(p.C, p.C_bs, a->C_stride);
    if (q.npl == 4) {
        switch (q.lanes) {
        case 1: return launch_full<T, 4, 1>(p, wide, st);
        case 2: return launch_full<T, 4, 2>(p, wide, st);
        case 4: return launch_full<T, 4, 4>(p, wide, st);
        case 8: return launch_full<T, 4, 8>(p, wide, st);
        default: return launch_full<T, 4, 16>(p, wide, st);
        }
    }
    if (q.npl == 8)
        return q.lanes == 1 ? launch_full<T, 8, 1>(p, wide, st) : launch_full<T, 8, 16>(p, wide, st);
    if (q.npl == 16)
        return q.lanes == 1 ? launch_full<T, 16, 1>(p, wide, st) : launch_full<T, 16, 16>(p, wide, st);
    return launch_full<T, 32, 1>(p, wide, st);
}

int check_sizes(const cnh_state_scan_args* a, const char* call) {
    CNH_CHECK(a != nullptr, -2, "%s: null arguments", call);
    if (int rc = check_float_type(a->dtype, call))
        return rc;
    CNH_CHECK(a->batch >= 0 && a->length >= 0 && a->channels >= 0, -2, "%s: batch %lld, length %lld, channels %lld", call,
              (long long)a->batch, (long long)a->length, (long long)a->channels);
    CNH_CHECK(a->states >= 1 && a->states <= 256, -3, "%s: %lld states; 1 to 256 are supported", call,
              (long long)a->states);
    CNH_CHECK(a->softplus == 0 || a->softplus == 1, -2, "%s: softplus %d is neither 0 nor 1", call, a->softplus);
    CNH_CHECK(a->batch < ((int64_t)1 << 31) && a->length < ((int64_t)1 << 31) && a->channels < ((int64_t)1 << 24), -3,
              "%s: batch %lld, length %lld (below 2^31), channels %lld (below 2^24)", call, (long long)a->batch,
              (long long)a->length, (long long)a->channels);
    return 0;
}

} // namespace

extern "C" int64_t cnh_state_scan_workspace(const cnh_state_scan_args* a) {
    if (int rc = check_sizes(a, "cnh_state_scan_workspace"))
        return rc;
    if (a->batch == 0 || a->channels == 0)
        return 0;
    return plan_of(a).bytes;
}

extern "C" int cnh_state_scan(const cnh_state_scan_args* a, cnh_stream s) {
    const char* call = "cnh_state_scan";
    if (int rc = check_sizes(a, call))
        return rc;
    if (a->batch == 0 || a->channels == 0 || (a->length == 0 && !a->state_out))
        return 0;
    CNH_CHECK(a->A && (a->length == 0 || (a->x && a->delta && a->B && a->C && a->y)), -2,
              "%s: null x, delta, A, B, C or y", call);
    const int esz = dtype_size(a->dtype);
    const int64_t D = a->channels, N = a->states;
    auto rows = [&](const char* what, const void* ptr, int64_t bs, int64_t st, int64_t cols) {
        return Extent{what, ptr, span_of(a->batch, bs, a->length, st, cols) * esz};
    };
    const __int128 state = (__int128)a->batch * D * N * esz;
    CNH_CHECK(state < ((__int128)1 << 62), -3, "%s: the states do not fit any memory", call);
    const Plan q = plan_of(a);
    const Extent y = rows("y", a->y, a->y_batch_stride, a->y_stride, D),
                 out{"state_out", a->state_out, (int64_t)state}, in{"state_in", a->state_in, (int64_t)state},
                 ws{"workspace", a->workspace, q.bytes}, len{"lengths", a->lengths, a->batch * 4};
    const Extent reads[] = {rows("x", a->x, a->x_batch_stride, a->x_stride, D),
                            rows("delta", a->delta, a->delta_batch_stride, a->delta_stride, D),
                            rows("z", a->z, a->z_batch_stride, a->z_stride, D),
                            rows("B", a->B, a->B_batch_stride, a->B_stride, N),
                            rows("C", a->C, a->C_batch_stride, a->C_stride, N),
                            {"A", a->A, D * N * esz},
                            {"skip", a->skip, D * esz},
                            {"delta_bias", a->delta_bias, D * esz}};
    for (const Extent* e : {&y, &out, &in})
        if (int rc = check_extent(*e, esz, call))
            return rc;
    for (const Extent& e : reads)
        if (int rc = check_extent(e, esz, call))
            return rc;
    if (int rc = check_extent(len, 4, call))
        return rc;
    if (a->length > 1)
        for (int64_t stride : {a->x_stride, a->delta_stride, a->z ? a->z_stride : 0, a->B_stride, a->C_stride, a->y_stride})
            CNH_CHECK(stride < ((int64_t)1 << 31) / esz, -3, "%s: %lld elements between tokens; rows are less than 2 GiB apart",
                      call, (long long)stride);
    CNH_CHECK(q.bytes == 0 || (a->workspace && a->workspace_bytes >= q.bytes), -2,
              "%s: a workspace of %lld bytes is needed, %lld given", call, (long long)q.bytes,
              (long long)(a->workspace ? a->workspace_bytes : 0));
    CNH_CHECK(q.bytes == 0 || aligned_to(a->workspace, 16), -2, "%s: the workspace is not aligned to 16 bytes", call);
    CNH_CHECK(a->length == 0 || rows_apart(a->batch, a->y_batch_stride, a->length, a->y_stride, D), -2,
              "%s: rows of y overlap", call);
    const Extent* writes[] = {&y, &out, &ws};
    for (const Extent* w : writes) {
        for (const Extent& e : reads)
            CNH_CHECK(!overlap(*w, e), -2, "%s: %s overlaps %s", call, w->what, e.what);
        CNH_CHECK(!overlap(*w, len), -2, "%s: %s overlaps lengths", call, w->what);
        CNH_CHECK(w == &out || !overlap(*w, in), -2, "%s: %s overlaps state_in", call, w->what);
        CNH_CHECK(w == &out || !overlap(*w, out), -2, "%s: %s overlaps state_out", call, w->what);
    }
    CNH_CHECK(!overlap(y, ws), -2, "%s: y overlaps the workspace", call);
    CNH_CHECK(!overlap(out, in) || out.ptr == in.ptr, -2, "%s: state_out overlaps state_in without being the same", call);
    if (int rc = ensure_init())
        return rc;
    DeviceScope dev;
    if (int rc = dev.enter())
        return rc;
    return a->dtype == CNH_F32 ? run<float>(a, q, as_stream(s)) : run<double>(a, q, as_stream(s));
}
