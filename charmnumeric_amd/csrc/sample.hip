// Draw of one word per row of logits, from a given random number:
//   w = exp((l - max l) / temperature);  top-k keeps the k largest (ties: the lowest indices), top-p the
//   shortest run of what is left, in descending order, whose mass reaches p of theirs, min-p those with
//   w >= min_p; the word is the first in descending order whose running mass passes u times the mass kept.
//
// Every cut keeps a prefix of the descending order, so a row needs no full sort: a histogram over the
// depth (max - l) / temperature finds the bin a cut or the draw falls into, and only that bin (or, when
// they are few, everything down to the cut) is gathered into shared memory and sorted. A bin that is too
// crowded for that is split by the bits of its values until it is small enough or one value.
//
// Masses are 64-bit integers, w in steps of 2^-45 (coarser beyond 2^17 words, so that a row's sum fits
// 62 bits): additions in any order give the same sum, so the histogram's atomics cannot change a result.
// A word 32 below the maximum (e^-32 < 2^-46) has no mass and is never drawn. Exponentials and depths are
// 64-bit whatever the logits' type: the drawn word changes where a running sum passes the random number.
//
// Bound by memory for many rows (one workgroup per row, the passes behind the first come from the
// caches) and by the length of one row's passes for few.
#include "sequence.h"

#include <algorithm>

using namespace cnh;

namespace {

constexpr int kThreads = 1024, kWaves = kThreads / 64, kBins = 2048, kList = 2048;
constexpr double kDepth = 32.0, kBinsPerUnit = kBins / kDepth;

template <typename T>
struct SampleParams {
    int64_t rows, vocab, stride;
    const T* logits;
    const double* u;
    double temperature, top_p, min_p;
    int top_k;
    const double* temperatures;
    const int32_t* top_ks;
    const double *top_ps, *min_ps;
    int32_t* out;
    double mass_scale; // mass of weight 1
};

template <typename T>
struct KeyOf;
template <>
struct KeyOf<float> {
    typedef uint32_t type;
};
template <>
struct KeyOf<double> {
    typedef uint64_t type;
};

// Integers in the order of the values; -0 and +0 are one value, NaN lies below everything.
__device__ __forceinline__ uint32_t key_of(float l) {
    if (l != l)
        return 0;
    const uint32_t b = __float_as_uint(l + 0.0f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ uint64_t key_of(double l) {
    if (l != l)
        return 0;
    const uint64_t b = (uint64_t)__double_as_longlong(l + 0.0);
    return b >> 63 ? ~b : b | (1ull << 63);
}
__device__ __forceinline__ float value_of(uint32_t k) {
    return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}
__device__ __forceinline__ double value_of(uint64_t k) {
    return __longlong_as_double((long long)(k >> 63 ? k & ~(1ull << 63) : ~k));
}

template <typename V>
__device__ __forceinline__ V shuffle_up(V v, int o) {
    return __shfl_up(v, o, 64);
}

template <typename T>
struct Shared {
    typedef typename KeyOf<T>::type Key;
    // the first histogram, as running sums including the bin itself once it is complete
    uint32_t count[kBins];
    unsigned long long mass[kBins];
    union {
        struct {
            Key key[kList];
            uint32_t index[kList];
            unsigned long long mass[kList];
        } list;
        struct {
            uint32_t count[kBins];
            unsigned long long mass[kBins];
        } sub;
    };
    unsigned long long wave_mass[kWaves];
    uint32_t wave_count[kWaves];
    Key wave_key[kWaves];
    uint32_t wave_index[kWaves];
    unsigned long long found_mass, found_before;
    uint32_t found, listed, found_count;
    Key low, high;
};

// One row's walk in descending order; all lanes of the workgroup go through it together.
template <typename T, int VEC>
struct Row {
    typedef typename KeyOf<T>::type Key;
    Shared<T>& sh;
    const T* logits;
    int64_t vocab;
    double top, inv; // largest logit, 1 / temperature
    double scale;
    int tid;

    __device__ __forceinline__ double depth(T l) const { return (double)l == top ? 0.0 : (top - (double)l) * inv; }
    __device__ __forceinline__ int bin_at(double d) const {
        return d < kDepth ? (int)(d * kBinsPerUnit) : kBins; // NaN: beyond the last bin as well
    }
    __device__ __forceinline__ double weight(double d) const { return exp(-d); }
    __device__ __forceinline__ unsigned long long mass_of(double w) const {
        return (unsigned long long)(w * scale + 0.5);
    }

    // f(logit, index) for every word; each lane meets its words in ascending order.
    template <typename F>
    __device__ __forceinline__ void sweep(F f) const {
        constexpr int AHEAD = 4;
        const int64_t packs = vocab / VEC;
        for (int64_t i0 = tid; i0 < packs; i0 += (int64_t)kThreads * AHEAD) {
            Pack<T, VEC> q[AHEAD];
#pragma unroll
            for (int a = 0; a < AHEAD; ++a)
                if (i0 + a * kThreads < packs)
                    load_pack(q[a], logits + (i0 + a * kThreads) * VEC);
#pragma unroll
            for (int a = 0; a < AHEAD; ++a)
                if (i0 + a * kThreads < packs) {
#pragma unroll
                    for (int j = 0; j < VEC; ++j)
                        f(q[a].v[j], (uint32_t)((i0 + a * kThreads) * VEC + j));
                }
        }
        if (VEC > 1)
            for (int64_t i = packs * VEC + tid; i < vocab; i += kThreads)
                f(logits[i], (uint32_t)i);
    }

    // Turns a histogram into running sums (each bin's own included). Two bins a lane.
    __device__ __forceinline__ void running_sums(uint32_t* count, unsigned long long* mass) {
        static_assert(kBins == 2 * kThreads, "two bins a lane");
        uint32_t c0 = count[2 * tid], c = c0 + count[2 * tid + 1];
        unsigned long long m0 = mass[2 * tid], m = m0 + mass[2 * tid + 1];
        const uint32_t c_own = c;
        const unsigned long long m_own = m;
        const int lane = tid & 63;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const uint32_t cu = shuffle_up(c, o);
            const unsigned long long mu = shuffle_up(m, o);
            if (lane >= o) {
                c += cu;
                m += mu;
            }
        }
        if (lane == 63) {
            sh.wave_count[tid >> 6] = c;
            sh.wave_mass[tid >> 6] = m;
        }
        __syncthreads();
        for (int w = 0; w < tid >> 6; ++w) {
            c += sh.wave_count[w];
            m += sh.wave_mass[w];
        }
        count[2 * tid] = c - c_own + c0;
        count[2 * tid + 1] = c;
        mass[2 * tid] = m - m_own + m0;
        mass[2 * tid + 1] = m;
        __syncthreads();
    }

    // The first bin whose end satisfies `done(count, mass)` (running sums, monotone), kBins if none.
    template <typename P>
    __device__ __forceinline__ uint32_t first_bin(const uint32_t* count, const unsigned long long* mass, P done) {
        if (tid == 0)
            sh.found = kBins;
        __syncthreads();
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int b = 2 * tid + j;
            if (done(count[b], mass[b]) && (b == 0 || !done(count[b - 1], mass[b - 1])))
                sh.found = b; // one lane at most
        }
        __syncthreads();
        const uint32_t b = sh.found;
        __syncthreads();
        return b;
    }

    __device__ __forceinline__ void clear(uint32_t* count, unsigned long long* mass) {
        count[2 * tid] = count[2 * tid + 1] = 0;
        mass[2 * tid] = mass[2 * tid + 1] = 0;
        __syncthreads();
    }

    // Words accepted by `take(logit)` into the list, in descending order (ties: ascending index) with
    // running masses. Returns how many; the caller knows that they fit.
    template <typename P>
    __device__ __forceinline__ uint32_t gather(P take) {
        if (tid == 0)
            sh.listed = 0;
        __syncthreads();
        sweep([&](T l, uint32_t i) {
            if (take(l)) {
                const uint32_t at = atomicAdd(&sh.listed, 1u);
                if (at < kList) {
                    sh.list.key[at] = key_of(l);
                    sh.list.index[at] = i;
                }
            }
        });
        __syncthreads();
        const uint32_t n = min(sh.listed, (uint32_t)kList);
        uint32_t size = 2;
        while (size < n)
            size *= 2;
        for (uint32_t i = n + tid; i < size; i += kThreads) {
            sh.list.key[i] = 0;
            sh.list.index[i] = 0xffffffffu;
        }
        __syncthreads();
        // bitonic sort, one pair a lane
        for (uint32_t run = 2; run <= size; run *= 2)
            for (uint32_t step = run / 2; step > 0; step /= 2) {
                const uint32_t a = 2 * tid - (tid & (step - 1)), b = a + step;
                if (b < size) {
                    const Key ka = sh.list.key[a], kb = sh.list.key[b];
                    const uint32_t ia = sh.list.index[a], ib = sh.list.index[b];
                    const bool before = ka > kb || (ka == kb && ia < ib);
                    if (before != ((a & run) == 0)) {
                        sh.list.key[a] = kb;
                        sh.list.key[b] = ka;
                        sh.list.index[a] = ib;
                        sh.list.index[b] = ia;
                    }
                }
                __syncthreads();
            }
        // running masses, two words a lane
        unsigned long long m0 = 0, m = 0;
        if (2 * tid < n)
            m0 = m = mass_of(weight(depth(value_of(sh.list.key[2 * tid]))));
        if (2 * tid + 1 < n)
            m += mass_of(weight(depth(value_of(sh.list.key[2 * tid + 1]))));
        const unsigned long long own = m;
        const int lane = tid & 63;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const unsigned long long mu = shuffle_up(m, o);
            if (lane >= o)
                m += mu;
        }
        if (lane == 63)
            sh.wave_mass[tid >> 6] = m;
        __syncthreads();
        for (int w = 0; w < tid >> 6; ++w)
            m += sh.wave_mass[w];
        if (2 * tid < kList) {
            sh.list.mass[2 * tid] = m - own + m0;
            sh.list.mass[2 * tid + 1] = m;
        }
        __syncthreads();
        return n;
    }

    // How many of the first n listed words do not satisfy `done(place, running mass)` (monotone).
    template <typename P>
    __device__ __forceinline__ uint32_t listed_before(uint32_t n, P done) {
        if (tid == 0)
            sh.found = n;
        __syncthreads();
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const uint32_t i = 2 * tid + j;
            if (i < n && done(i) && (i == 0 || !done(i - 1)))
                sh.found = i;
        }
        __syncthreads();
        const uint32_t i = sh.found;
        __syncthreads();
        return i;
    }

    // The first word in descending order at whose end `done(count, mass)` holds, found in the completed
    // first histogram; its running mass, and its index when `want_index`.
    template <typename P>
    __device__ __forceinline__ void descend(P done, bool want_index, unsigned long long* mass, uint32_t* index) {
        const uint32_t b = first_bin(sh.count, sh.mass, done);
        uint32_t base_count = b ? sh.count[b - 1] : 0;
        unsigned long long base_mass = b ? sh.mass[b - 1] : 0;
        uint32_t n = sh.count[b] - base_count;
        Key high = 0, low = 0;
        if (n <= kList) {
            n = gather([&](T l) { return bin_at(depth(l)) == (int)b; });
        } else {
            // the range of the crowded bin's values
            Key hi = 0, lo = ~(Key)0;
            sweep([&](T l, uint32_t) {
                if (bin_at(depth(l)) == (int)b) {
                    const Key k = key_of(l);
                    hi = k > hi ? k : hi;
                    lo = k < lo ? k : lo;
                }
            });
            if (tid == 0) {
                sh.high = 0;
                sh.low = ~(Key)0;
            }
            __syncthreads();
            if constexpr (sizeof(Key) == 8) {
                atomicMax((unsigned long long*)&sh.high, (unsigned long long)hi);
                atomicMin((unsigned long long*)&sh.low, (unsigned long long)lo);
            } else {
                atomicMax((uint32_t*)&sh.high, (uint32_t)hi);
                atomicMin((uint32_t*)&sh.low, (uint32_t)lo);
            }
            __syncthreads();
            high = sh.high;
            low = sh.low;
            __syncthreads();
            while (n > kList && low < high) {
                int width = 0; // bits of high - low
                for (Key r = high - low; r; r >>= 1)
                    ++width;
                const int shift = width > 11 ? width - 11 : 0;
                clear(sh.sub.count, sh.sub.mass);
                sweep([&](T l, uint32_t) {
                    const Key k = key_of(l);
                    if (k >= low && k <= high) {
                        const uint32_t s = (uint32_t)((high - k) >> shift);
                        atomicAdd(&sh.sub.count[s], 1u);
                        atomicAdd(&sh.sub.mass[s], mass_of(weight(depth(l))));
                    }
                });
                __syncthreads();
                running_sums(sh.sub.count, sh.sub.mass);
                const uint32_t s = first_bin(sh.sub.count, sh.sub.mass, [&](uint32_t c, unsigned long long m) {
                    return done(base_count + c, base_mass + m);
                });
                n = sh.sub.count[s] - (s ? sh.sub.count[s - 1] : 0);
                if (s) {
                    base_count += sh.sub.count[s - 1];
                    base_mass += sh.sub.mass[s - 1];
                }
                high -= (Key)s << shift;
                const Key span = ((Key)1 << shift) - 1;
                low = high - low > span ? high - span : low;
                __syncthreads();
            }
            if (n > kList) {
                // words of one value: the place follows from their common mass
                const unsigned long long each = mass_of(weight(depth(value_of(high))));
                uint32_t lo_j = 1, hi_j = n;
                while (lo_j < hi_j) {
                    const uint32_t mid = lo_j + (hi_j - lo_j) / 2;
                    if (done(base_count + mid, base_mass + mid * each))
                        hi_j = mid;
                    else
                        lo_j = mid + 1;
                }
                *mass = base_mass + lo_j * each;
                if (want_index)
                    *index = nth_of_value(high, lo_j);
                return;
            }
            n = gather([&](T l) {
                const Key k = key_of(l);
                return k >= low && k <= high;
            });
        }
        const uint32_t i = min(
            listed_before(n, [&](uint32_t j) { return done(base_count + j + 1, base_mass + sh.list.mass[j]); }), n - 1);
        *mass = base_mass + sh.list.mass[i];
        *index = sh.list.index[i];
        __syncthreads();
    }

    // Index of the nth word (from 1, in ascending order) whose value has this key.
    __device__ __forceinline__ uint32_t nth_of_value(Key k, uint32_t nth) {
        uint32_t seen = 0;
        if (tid == 0)
            sh.found = 0xffffffffu;
        __syncthreads();
        for (int64_t i0 = 0; i0 < vocab; i0 += kThreads) {
            const int64_t i = i0 + tid;
            const bool hit = i < vocab && key_of(logits[i]) == k;
            const unsigned long long ballot = __ballot(hit);
            if ((tid & 63) == 0)
                sh.wave_count[tid >> 6] = (uint32_t)__popcll(ballot);
            __syncthreads();
            uint32_t before = seen, all = seen;
            for (int w = 0; w < kWaves; ++w) {
                if (w < tid >> 6)
                    before += sh.wave_count[w];
                all += sh.wave_count[w];
            }
            if (hit && before + (uint32_t)__popcll(ballot & ((1ull << (tid & 63)) - 1)) + 1 == nth)
                sh.found = (uint32_t)i;
            seen = all;
            __syncthreads();
            if (seen >= nth)
                break;
        }
        const uint32_t at = sh.found;
        __syncthreads();
        return at;
    }
};

template <typename T, int VEC>
__global__ __launch_bounds__(kThreads) void sample_kernel(SampleParams<T> p) {
    typedef typename KeyOf<T>::type Key;
    __shared__ Shared<T> sh;
    const int tid = threadIdx.x;
    for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
        Row<T, VEC> r{sh, p.logits + row * p.stride, p.vocab, 0.0, 0.0, p.mass_scale, tid};
        const double temperature = p.temperatures ? p.temperatures[row] : p.temperature;
        const double top_p = p.top_ps ? p.top_ps[row] : p.top_p;
        double min_p = p.min_ps ? p.min_ps[row] : p.min_p;
        min_p = min_p > 0.0 ? fmin(min_p, 1.0) : 0.0;
        const int64_t top_k = p.top_ks ? p.top_ks[row] : p.top_k;

        // the largest logit and the lowest index that has it
        Key best = 0;
        uint32_t at = 0xffffffffu;
        r.sweep([&](T l, uint32_t i) {
            const Key k = key_of(l);
            if (k > best || (k == best && i < at)) {
                best = k;
                at = i;
            }
        });
#pragma unroll
        for (int o = 32; o >= 1; o >>= 1) {
            const Key k = (Key)__shfl_xor(best, o, 64);
            const uint32_t i = __shfl_xor(at, o, 64);
            if (k > best || (k == best && i < at)) {
                best = k;
                at = i;
            }
        }
        if ((tid & 63) == 0) {
            sh.wave_key[tid >> 6] = best;
            sh.wave_index[tid >> 6] = at;
        }
        __syncthreads();
        for (int w = 0; w < kWaves; ++w) {
            const Key k = sh.wave_key[w];
            const uint32_t i = sh.wave_index[w];
            if (k > best || (k == best && i < at)) {
                best = k;
                at = i;
            }
        }
        int32_t drawn = (int32_t)at;
        if (best <= key_of(-std::numeric_limits<T>::infinity())) {
            drawn = -1; // every word is masked (or no number)
        } else if (temperature > 0.0 && top_k != 1 && !(top_p <= 0.0)) {
            r.top = (double)value_of(best);
            r.inv = fmin(1.0 / temperature, std::numeric_limits<double>::max());
            const double u0 = p.u[row], u = u0 > 0.0 ? fmin(u0, 1.0) : 0.0;
            // The cut of a small top-k comes from counts alone, everything it keeps fits the list, and
            // the words' masses are formed for the listed ones only. Other rows weigh every word.
            bool weigh = !(top_k > 0 && top_k <= kList / 2);
            unsigned long long kept_by_min_p = 0, total = 0;
            uint32_t last = kBins;  // last bin of the list
            for (;;) {
                r.clear(sh.count, sh.mass);
                unsigned long long own = 0;
                if (weigh) {
                    r.sweep([&](T l, uint32_t) {
                        const double d = r.depth(l);
                        const int b = r.bin_at(d);
                        if (b < kBins) {
                            const double w = r.weight(d);
                            const unsigned long long m = r.mass_of(w);
                            atomicAdd(&sh.count[b], 1u);
                            atomicAdd(&sh.mass[b], m);
                            own += w >= min_p ? m : 0;
                        }
                    });
                } else {
                    r.sweep([&](T l, uint32_t) {
                        const int b = r.bin_at(r.depth(l));
                        if (b < kBins)
                            atomicAdd(&sh.count[b], 1u);
                    });
                }
                __syncthreads();
                r.running_sums(sh.count, sh.mass);
                const uint32_t words = sh.count[kBins - 1];
                total = sh.mass[kBins - 1];
                uint32_t by_k = kBins, by_p = kBins, by_min_p = kBins;
                if (top_k > 0 && top_k < (int64_t)words)
                    by_k = r.first_bin(sh.count, sh.mass, [&](uint32_t c, unsigned long long) { return c >= top_k; });
                if (weigh && top_p < 1.0) {
                    const double want = top_p * (double)total;
                    by_p = r.first_bin(sh.count, sh.mass,
                                       [&](uint32_t, unsigned long long m) { return (double)m >= want; });
                }
                if (min_p > 0.0)
                    by_min_p = (uint32_t)fmin(-log(min_p) * kBinsPerUnit + 1.0, (double)kBins); // one to spare
                last = min(min(by_k, by_p), by_min_p);
                // p of what top-k leaves needs all of that in the list
                if (top_p < 1.0 && top_k > 0 && (!weigh || by_k != kBins))
                    last = by_k;
                last = min(last, (uint32_t)kBins - 1);
                const uint32_t words_listed = sh.count[last];
                if (weigh) {
                    // sum of `own` over the workgroup
#pragma unroll
                    for (int o = 32; o >= 1; o >>= 1)
                        own += __shfl_xor(own, o, 64);
                    if ((tid & 63) == 0)
                        sh.wave_mass[tid >> 6] = own;
                    __syncthreads();
                    kept_by_min_p = 0;
                    for (int w = 0; w < kWaves; ++w)
                        kept_by_min_p += sh.wave_mass[w];
                    __syncthreads();
                }
                if (words_listed <= kList) {
                    const uint32_t n = r.gather([&](T l) { return r.bin_at(r.depth(l)) <= (int)last; });
                    uint32_t cut = top_k > 0 ? (uint32_t)min((int64_t)n, top_k) : n;
                    if (top_p < 1.0) {
                        // without a top-k that cuts, the list may end before the last word that counts
                        const unsigned long long of = weigh && by_k == kBins ? total : sh.list.mass[cut - 1];
                        const double want = top_p * (double)of;
                        cut = min(cut, r.listed_before(n, [&](uint32_t i) { return (double)sh.list.mass[i] >= want; }) + 1);
                    }
                    if (min_p > 0.0)
                        cut = min(cut, r.listed_before(n, [&](uint32_t i) {
                            return !(r.weight(r.depth(value_of(sh.list.key[i]))) >= min_p);
                        }));
                    const unsigned long long kept = sh.list.mass[cut - 1];
                    const unsigned long long target = min((unsigned long long)(u * (double)kept), kept - 1);
                    const uint32_t i =
                        r.listed_before(cut, [&](uint32_t j) { return sh.list.mass[j] > target; });
                    drawn = (int32_t)sh.list.index[min(i, cut - 1)];
                    break;
                }
                if (weigh) {
                    uint32_t index = 0;
                    unsigned long long of = total;
                    if (by_k != kBins)
                        r.descend([&](uint32_t c, unsigned long long) { return c >= top_k; }, false, &of, &index);
                    unsigned long long kept = of;
                    if (top_p < 1.0) {
                        const double want = top_p * (double)of;
                        r.descend([&](uint32_t, unsigned long long m) { return (double)m >= want; }, false, &kept,
                                  &index);
                        kept = min(kept, of);
                    }
                    if (min_p > 0.0)
                        kept = min(kept, kept_by_min_p);
                    const unsigned long long target = min((unsigned long long)(u * (double)kept), kept - 1);
                    r.descend([&](uint32_t, unsigned long long m) { return m > target; }, true, &kept, &index);
                    drawn = (int32_t)index;
                    break;
                }
                weigh = true; // a crowd at the cut: weigh every word and walk down to it
            }
        }
        if (tid == 0)
            p.out[row] = drawn;
        __syncthreads(); // the next row writes the shared memory again
    }
}

template <typename T>
int run(const cnh_sample_tokens_args* a, hipStream_t st) {
    SampleParams<T> p;
    p.rows = a->rows;
    p.vocab = a->vocab;
    p.stride = a->stride;
    p.logits = static_cast<const T*>(a->logits);
    p.u = a->u;
    p.temperature = a->temperature;
    p.top_p = a->top_p;
    p.min_p = a->min_p;
    p.top_k = a->top_k;
    p.temperatures = a->temperatures;
    p.top_ks = a->top_ks;
    p.top_ps = a->top_ps;
    p.min_ps = a->min_ps;
    p.out = a->out;
    int bits = 0; // ceil(log2(vocab))
    while (((int64_t)1 << bits) < a->vocab)
        ++bits;
    p.mass_scale = (double)((uint64_t)1 << std::min(45, 62 - bits));
    constexpr int W = Wide<T>::n;
    const unsigned groups = (unsigned)std::min<int64_t>(p.rows, 1 << 20);
    if (aligned_to(p.logits, 16) && (p.rows == 1 || p.stride % W == 0))
        sample_kernel<T, W><<<groups, kThreads, 0, st>>>(p);
    else
        sample_kernel<T, 1><<<groups, kThreads, 0, st>>>(p);
    CNH_HIP(hipGetLastError());
    return 0;
}

int check(const cnh_sample_tokens_args* a, const char* call) {
    CNH_CHECK(a != nullptr, -2, "%s: null arguments", call);
    if (int rc = check_float_type(a->dtype, call))
        return rc;
    CNH_CHECK(a->rows >= 0 && a->rows < ((int64_t)1 << 31), -3, "%s: %lld rows (0 to 2^31 - 1)", call, (long long)a->rows);
    CNH_CHECK(a->vocab >= 1 && a->vocab <= (1 << 22), -3, "%s: %lld words; 1 to 2^22 are supported", call,
              (long long)a->vocab);
    return 0;
}

} // namespace

extern "C" int64_t cnh_sample_tokens_workspace(const cnh_sample_tokens_args* a) {
    return check(a, "cnh_sample_tokens_workspace");
}

extern "C" int cnh_sample_tokens(const cnh_sample_tokens_args* a, cnh_stream s) {
    const char* call = "cnh_sample_tokens";
    if (int rc = check(a, call))
        return rc;
    if (a->rows == 0)
        return 0;
    CNH_CHECK(a->logits && a->u && a->out, -2, "%s: null logits, u or out", call);
    CNH_CHECK(a->temperatures || a->temperature >= 0.0, -2, "%s: temperature %g is negative or no number", call,
              a->temperature);
    CNH_CHECK(a->top_ks || a->top_k >= 0, -2, "%s: top_k %d is negative", call, a->top_k);
    CNH_CHECK(a->top_ps || a->top_p >= 0.0, -2, "%s: top_p %g is negative or no number", call, a->top_p);
    CNH_CHECK(a->min_ps || (a->min_p >= 0.0 && a->min_p <= 1.0), -2, "%s: min_p %g is not in [0, 1]", call, a->min_p);
    const int esz = dtype_size(a->dtype);
    const Extent logits{"logits", a->logits, span_of(1, 0, a->rows, a->stride, a->vocab) * esz},
        out{"out", a->out, a->rows * 4}, ks{"top_ks", a->top_ks, a->rows * 4};
    const Extent doubles[] = {{"u", a->u, a->rows * 8},
                              {"temperatures", a->temperatures, a->rows * 8},
                              {"top_ps", a->top_ps, a->rows * 8},
                              {"min_ps", a->min_ps, a->rows * 8}};
    if (int rc = check_extent(logits, esz, call))
        return rc;
    for (const Extent* e : {&out, &ks})
        if (int rc = check_extent(*e, 4, call))
            return rc;
    for (const Extent& e : doubles) {
        if (int rc = check_extent(e, 8, call))
            return rc;
        CNH_CHECK(!overlap(out, e), -2, "%s: out overlaps %s", call, e.what);
    }
    CNH_CHECK(!overlap(out, logits) && !overlap(out, ks), -2, "%s: out overlaps logits or top_ks", call);
    if (int rc = ensure_init())
        return rc;
    DeviceScope dev;
    if (int rc = dev.enter())
        return rc;
    return a->dtype == CNH_F32 ? run<float>(a, as_stream(s)) : run<double>(a, as_stream(s));
}
