// Draw of one word per row of logits, from a given random number:
//   w = exp((l - max l) / temperature);  top-k keeps the k largest (ties: the lowest indices), top-p the
//   shortest run of what is left, in descending order, whose mass reaches p of theirs, min-p those with
//   w >= min_p; the word is the first in descending order whose running mass passes u times the mass kept.
//
// Every cut keeps a prefix of the descending order, so a row needs no full sort: a histogram over the
// depth (max - l) / temperature finds the bin a cut or the draw falls into, and only that bin (or, when
// they are few, everything down to the cut) is gathered into shared memory and sorted there, by buckets
// and by counting inside a bucket. A bin that is too crowded for that is split by the bits of its values
// until it is small enough or one value.
//
// A small top-k needs no histogram of the row: the k-th largest of the lanes' own maxima, which the pass
// for the maximum has left behind, is at most the k-th largest word, so what is not below it (its bin)
// holds all that top-k keeps and little else. Two passes over the row, no exponential outside the list.
//
// Masses are 64-bit integers, w in steps of 2^-45 (coarser beyond 2^17 words, so that a row's sum fits
// 62 bits): additions in any order give the same sum, so the histogram's atomics cannot change a result.
// A word 32 below the maximum (e^-32 < 2^-46) has no mass and is never drawn. Exponentials and depths are
// 64-bit whatever the logits' type: the drawn word changes where a running sum passes the random number.
//
// Few rows whose every word has to be weighed are cut into slices: a pass for the slices' maxima, one that
// adds their weights up bin by bin in the workspace, and the row's own workgroup goes on from there.
//
// A row is one workgroup's, on one CU: what bounds it is that CU's rate of reading (two sweeps of a greedy draw over
// rows of 64 K to 256 K fp32 words: 150 GB/s, out of its L2; 80 to 105 GB/s over rows of 0.5 to 4 M words), the
// 64-bit arithmetic of the weighing, and some twenty short phases that each wait for their instructions. One row of
// 131072 fp32 words with a top-k of 50: 17.5 us, 7 of them its two sweeps. 256 rows of 50021, settings mixed:
// 34.4 us, the time of a row that has to be weighed; 256 of 1000 words, sorted whole: 12.0 us. One row of 131072
// without a top-k, in 16 slices: 4 + 6 + 20 us, with a top-p of 0.95 5 + 5 + 26.
#include "sequence.h"

#include <algorithm>
#include <limits>

using namespace cnh;

namespace {

constexpr int kThreads = 1024, kWaves = kThreads / 64, kBins = 2048, kList = kThreads;
constexpr double kDepth = 32.0, kBinsPerUnit = kBins / kDepth;

template <typename T>
struct SampleParams {
    int64_t rows, vocab, stride;
    int64_t first_row; // of this launch
    const T* logits;
    const double* u;
    double temperature, top_p, min_p;
    int top_k;
    const double* temperatures;
    const int32_t* top_ks;
    const double *top_ps, *min_ps;
    int32_t* out;
    double mass_scale; // mass of weight 1
    // Few rows: each is cut into slices that other workgroups weigh first. One entry per slice, per bin
    // or per row, rows one behind the other.
    int slices;
    int64_t slice; // words, a multiple of what a 16-byte access takes
    T* tops;
    unsigned long long *masses, *above;
    uint32_t* counts;
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

// A row's phases run once each, so what they cost besides memory is mostly the fetching of their
// instructions: sums and maxima over the lanes by row operations are few of them.

// Sums over the lanes of a row of 16 up to this one; of a wavefront.
template <typename V>
__device__ __forceinline__ V row_sums(V v) {
    v += moved<0x111, 0xf>(v); // row_shr 1, 2, 4, 8
    v += moved<0x112, 0xf>(v);
    v += moved<0x114, 0xf>(v);
    v += moved<0x118, 0xf>(v);
    return v;
}
template <typename V>
__device__ __forceinline__ V wave_sums(V v) {
    v = row_sums(v);
    v += moved<0x142, 0xa>(v); // row_bcast 15 to the odd rows
    v += moved<0x143, 0xc>(v); // row_bcast 31 to the upper two
    return v;
}
// The largest value of a row of 16, in all its lanes; of a wavefront.
template <typename V>
__device__ __forceinline__ V larger(V a, V b) { return b > a ? b : a; }
template <typename V>
__device__ __forceinline__ V row_max(V v) {
    v = larger(v, moved<0xB1, 0xf>(v));  // quad_perm [1,0,3,2]
    v = larger(v, moved<0x4E, 0xf>(v));  // quad_perm [2,3,0,1]
    v = larger(v, moved<0x141, 0xf>(v)); // row_half_mirror
    v = larger(v, moved<0x140, 0xf>(v)); // row_mirror
    return v;
}
template <typename V>
__device__ __forceinline__ V wave_max(V v) {
    v = row_max(v);
    return larger(larger(of_lane(v, 0), of_lane(v, 16)), larger(of_lane(v, 32), of_lane(v, 48)));
}

template <typename T>
struct Shared {
    typedef typename KeyOf<T>::type Key;
    // the first histogram, as running sums including the bin itself once it is complete
    // (bin kBins takes what lies beyond, with no mass)
    uint32_t count[kBins + 2];
    unsigned long long mass[kBins + 2];
    double level[kBins + 2]; // e^-(bin's depth)
    union {
        struct {
            Key key[kList];
            uint32_t index[kList];
            unsigned long long mass[kList];
            Key grouped_key[kList];
            uint32_t grouped_index[kList];
            uint32_t start[kList + 1]; // of each bucket
        } list;
        struct {
            uint32_t count[kBins];
            unsigned long long mass[kBins];
        } sub;
    };
    unsigned long long wave_mass[kWaves];
    uint32_t wave_count[kWaves];
    T wave_top[kWaves];
    uint32_t found, listed;
    Key low, high;
};

// What ends a run of the descending order: a number of words, a mass reached, or a mass passed.
struct Until {
    enum Kind { COUNT, REACHED, PASSED } kind;
    uint32_t words;
    double reached;
    unsigned long long passed;
    __device__ __forceinline__ bool operator()(uint32_t count, unsigned long long mass) const {
        return kind == COUNT ? count >= words : kind == REACHED ? (double)mass >= reached : mass > passed;
    }
};

// Which words a list takes: those of bins b0 to b1 and of bin b2, or (keyed) those with keys low to high.
template <typename Key>
struct Range {
    uint32_t b0, b1, b2;
    bool keyed;
    Key low, high;
};

// One row's walk in descending order; all lanes of the workgroup go through it together.
template <typename T>
struct Row {
    typedef typename KeyOf<T>::type Key;
    Shared<T>& sh;
    const T* logits;
    int64_t vocab;
    double top, inv; // largest logit (finite), 1 / temperature
    double scale;
    int tid;

    __device__ __forceinline__ void set(T largest, double temperature) {
        top = (double)largest;
        inv = fmin(1.0 / temperature, std::numeric_limits<double>::max());
    }
    // (max - l) / temperature; no number for NaN
    __device__ __forceinline__ double depth(T l) const { return (top - (double)l) * inv; }
    // The nearest bin (bin b is at depth b / kBinsPerUnit), kBins for what is deeper than the last and
    // for NaN. Adding 1.5 x 2^52 leaves the rounded integer in the low bits of the sum. Every step is
    // monotone, so bins are.
    __device__ __forceinline__ static int bin_at(double d, double* rest = nullptr) {
        const double t = fma(d, kBinsPerUnit, 0x1.8p52);
        if (rest)
            *rest = fma(t - 0x1.8p52, -1.0 / kBinsPerUnit, d);
        return d <= (kBins - 1) / kBinsPerUnit ? __double2loint(t) : kBins;
    }
    __device__ __forceinline__ int bin_of(T l) const { return bin_at(depth(l)); }
    // Logits that the words of bin b0 to b1 lie between, with some room: what a pass tests first.
    struct Between {
        T low, high;
        __device__ __forceinline__ bool has(T l) const { return l >= low && l <= high; }
    };
    __device__ __forceinline__ Between between(uint32_t b0, uint32_t b1) const {
        const double room = 16.0 * (double)std::numeric_limits<T>::epsilon(), step = 1.0 / kBinsPerUnit / inv;
        const double far = (b1 + 0.5) * step, near = (b0 - 0.5) * step;
        return {(T)(top - (far + fabs(top)) * room - far),
                b0 == 0 ? std::numeric_limits<T>::infinity() : (T)(top + (far + fabs(top)) * room - near)};
    }
    // e^-depth: the level of the bin times e^-r of the rest, |r| <= 2^-7 (r^6 / 6! is 2^-51 of it).
    __device__ __forceinline__ double weight_at(int bin, double r) const {
        double e = -1.0 / 120;
        e = fma(e, r, 1.0 / 24);
        e = fma(e, r, -1.0 / 6);
        e = fma(e, r, 0.5);
        e = fma(e, r, -1.0);
        e = fma(e, r, 1.0);
        return e * sh.level[bin];
    }
    bool weighed; // by weight_at(), which the list then goes by as well; the levels are there
    __device__ __forceinline__ double weight(T l) const {
        double r;
        const double d = depth(l);
        const int bin = bin_at(d, &r);
        return weighed ? weight_at(bin, r) : bin < kBins ? exp(-d) : 0.0;
    }
    __device__ __forceinline__ void fill_levels() const {
        for (int b = tid; b <= kBins; b += kThreads)
            sh.level[b] = b < kBins ? exp(-b / kBinsPerUnit) : 0.0;
    }
    // w * scale below 2^52: adding 2^52 leaves the rounded integer in the low bits
    __device__ __forceinline__ unsigned long long mass_of(double w) const {
        return (unsigned long long)__double_as_longlong(fma(w, scale, 0x1p52)) & 0xfffffffffffffull;
    }

    // f(pack, index of its first word) for every word: 16-byte packs from the first aligned one on, AHEAD
    // of a lane at once, and what is before the first and behind the last whole one as packs of one.
    template <typename F>
    __device__ __forceinline__ void sweep(F f) const {
        constexpr int VEC = Wide<T>::n, AHEAD = 2;
        const uint32_t words = (uint32_t)vocab;
        const uint32_t head = min((uint32_t)((16 - ((uintptr_t)logits & 15)) & 15) / (uint32_t)sizeof(T), words);
        const uint32_t packs = (words - head) / VEC;
        const T* base = logits + head;
        uint32_t i0 = 0;
        for (; i0 + AHEAD * kThreads <= packs; i0 += AHEAD * kThreads) {
            Pack<T, VEC> q[AHEAD];
#pragma unroll
            for (int a = 0; a < AHEAD; ++a)
                load_pack(q[a], base + (int64_t)(i0 + a * kThreads + tid) * VEC);
#pragma unroll
            for (int a = 0; a < AHEAD; ++a)
                f(q[a], head + (i0 + a * kThreads + tid) * VEC);
        }
        for (uint32_t i = i0 + tid; i < packs; i += kThreads) {
            Pack<T, VEC> q;
            load_pack(q, base + (int64_t)i * VEC);
            f(q, head + i * VEC);
        }
        const uint32_t tail = head + packs * VEC, single = head + (words - tail); // at most 2 (VEC - 1)
        if ((uint32_t)tid < single) {
            const uint32_t i = (uint32_t)tid < head ? (uint32_t)tid : tail + ((uint32_t)tid - head);
            Pack<T, 1> q;
            q.v[0] = logits[i];
            f(q, i);
        }
    }
    // f(logit, index) for the words that `test` lets through: in most packs of a row it is none.
    template <typename P, typename F>
    __device__ __forceinline__ void sweep_some(P test, F f) const {
        sweep([&](const auto& q, uint32_t i) {
            constexpr int N = (int)(sizeof(q.v) / sizeof(T));
            bool any = false;
#pragma unroll
            for (int j = 0; j < N; ++j)
                any |= test(q.v[j]);
            if (any)
#pragma unroll
                for (int j = 0; j < N; ++j)
                    if (test(q.v[j]))
                        f(q.v[j], i + j);
        });
    }

    // Sum of v over the lanes up to this one, of the whole workgroup.
    template <typename V>
    __device__ __forceinline__ V running_sum(V v, V* waves) const {
        static_assert(kWaves == 16, "a row of lanes");
        v = wave_sums(v);
        const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
        if ((tid & 63) == 63)
            waves[wave] = v;
        __syncthreads();
        const V upto = row_sums(waves[tid & 15]);
        return wave ? v + of_lane(upto, wave - 1) : v;
    }
    // Turns a histogram into running sums (each bin's own included). Two bins a lane.
    __device__ __forceinline__ void running_sums(uint32_t* count, unsigned long long* mass) {
        static_assert(kBins == 2 * kThreads, "two bins a lane");
        const uint32_t c1 = count[2 * tid + 1], c = running_sum(count[2 * tid] + c1, sh.wave_count);
        const unsigned long long m1 = mass[2 * tid + 1], m = running_sum(mass[2 * tid] + m1, sh.wave_mass);
        count[2 * tid] = c - c1;
        count[2 * tid + 1] = c;
        mass[2 * tid] = m - m1;
        mass[2 * tid + 1] = m;
        __syncthreads();
    }

    // The first bin whose end satisfies `done(count, mass)` (running sums, monotone), kBins if none.
    template <typename P>
    __device__ __forceinline__ uint32_t first_bin(const uint32_t* count, const unsigned long long* mass, P done) {
        if (tid == 0)
            sh.found = kBins;
        __syncthreads();
        if (first_lane(done(count[2 * tid + 1], mass[2 * tid + 1])))
            atomicMin(&sh.found, done(count[2 * tid], mass[2 * tid]) ? 2 * tid : 2 * tid + 1);
        __syncthreads();
        const uint32_t b = sh.found;
        __syncthreads();
        return b;
    }
    // Is this the first lane of its wavefront with `yes`?
    __device__ __forceinline__ bool first_lane(bool yes) const {
        return yes && __ffsll(__ballot(yes)) - 1 == (tid & 63);
    }

    __device__ __forceinline__ void clear(uint32_t* count, unsigned long long* mass) {
        count[2 * tid] = count[2 * tid + 1] = 0;
        mass[2 * tid] = mass[2 * tid + 1] = 0;
        __syncthreads();
    }

    // The words of a range into the list, in descending order (ties: ascending index) with running masses.
    // Returns how many there are; beyond kList the list is of no use.
    __device__ __forceinline__ uint32_t gather(const Range<Key>& g) {
        sh.list.start[tid] = 0;
        if (tid == 0)
            sh.listed = 0;
        __syncthreads();
        auto put = [&](T l, uint32_t i) {
            const uint32_t at = atomicAdd(&sh.listed, 1u);
            if (at < kList) {
                sh.list.key[at] = key_of(l);
                sh.list.index[at] = i;
            }
        };
        const Between first = between(g.b0, g.b1), second = between(g.b2, g.b2);
        auto look = [&](auto maybe) {
            sweep_some(maybe, [&](T l, uint32_t i) {
                bool take;
                if (g.keyed) {
                    const Key k = key_of(l);
                    take = k >= g.low && k <= g.high;
                } else {
                    const uint32_t b = (uint32_t)bin_of(l);
                    take = (b >= g.b0 && b <= g.b1) || b == g.b2;
                }
                if (take)
                    put(l, i);
            });
        };
        if (g.b0 == 0 && g.b1 == g.b2) // one comparison tells
            look([&](T l) { return l >= first.low; });
        else
            look([&](T l) { return first.has(l) || second.has(l); });
        __syncthreads();
        const uint32_t n = sh.listed;
        if (n > kList) {
            __syncthreads();
            return n;
        }
        // one word a lane from here on: into its bucket (equal steps of the depth, or of the key), ...
        const int shift = g.keyed ? max(bits_of(g.high - g.low) - 10, 0) : 0;
        const double from = g.b0 - 0.5, per = (double)kList / (max(g.b1, g.b2) + 1 - g.b0);
        const bool own = tid < n;
        Key key = 0;
        uint32_t index = 0, group = 0, slot = 0;
        if (own) {
            key = sh.list.key[tid];
            index = sh.list.index[tid];
            group = g.keyed ? (uint32_t)((g.high - key) >> shift)
                            : min((uint32_t)fmax((depth(value_of(key)) * kBinsPerUnit - from) * per, 0.0),
                                  (uint32_t)kList - 1);
            slot = atomicAdd(&sh.list.start[group], 1u);
        }
        __syncthreads();
        const uint32_t size = sh.list.start[tid];
        const uint32_t upto = running_sum(size, sh.wave_count); // ends in a barrier behind the loads of `size`
        sh.list.start[tid] = upto - size;
        if (tid == kThreads - 1)
            sh.list.start[kList] = upto;
        __syncthreads();
        uint32_t begin = 0, end = 0;
        if (own) {
            begin = sh.list.start[group];
            end = sh.list.start[group + 1];
            sh.list.grouped_key[begin + slot] = key;
            sh.list.grouped_index[begin + slot] = index;
        }
        __syncthreads();
        // ... and to its place in it, which the words before it in the order leave free
        uint32_t place = begin;
        for (uint32_t q = begin; q < end; ++q) {
            const Key k = sh.list.grouped_key[q];
            place += k > key || (k == key && sh.list.grouped_index[q] < index);
        }
        if (own) {
            sh.list.key[place] = key;
            sh.list.index[place] = index;
        }
        __syncthreads();
        const unsigned long long m = own ? mass_of(weight(value_of(sh.list.key[tid]))) : 0;
        sh.list.mass[tid] = running_sum(m, sh.wave_mass);
        __syncthreads();
        return n;
    }

    // How many of the first n listed words come before the first that satisfies `done(place)`.
    template <typename P>
    __device__ __forceinline__ uint32_t listed_before(uint32_t n, P done) {
        if (tid == 0)
            sh.found = n;
        __syncthreads();
        if (first_lane(tid < n && done(tid)))
            atomicMin(&sh.found, (uint32_t)tid);
        __syncthreads();
        const uint32_t i = sh.found;
        __syncthreads();
        return i;
    }

    __device__ __forceinline__ static int bits_of(Key v) {
        return v == 0 ? 0 : sizeof(Key) == 8 ? 64 - __clzll((unsigned long long)v) : 32 - __clz((int)v);
    }
    // Splits a bin that is too crowded for the list by the bits of its values until the part with the
    // first word at whose end `done` holds fits it, or is a single value. g: the bin, then the part;
    // count, mass: what is in front of the bin, then of the part. Returns the part's words.
    __device__ __forceinline__ uint32_t narrow(Range<Key>& g, const Until& done, uint32_t& count, unsigned long long& mass) {
        const Between near = between(g.b2, g.b2);
        auto test = [&](T l) { return near.has(l); };
        if (tid == 0) {
            sh.high = 0;
            sh.low = ~(Key)0;
        }
        __syncthreads();
        Key high = 0, low = ~(Key)0;
        sweep_some(test, [&](T l, uint32_t) {
            if (bin_of(l) == (int)g.b2) {
                const Key k = key_of(l);
                high = k > high ? k : high;
                low = k < low ? k : low;
            }
        });
        if constexpr (sizeof(Key) == 8) {
            atomicMax((unsigned long long*)&sh.high, (unsigned long long)high);
            atomicMin((unsigned long long*)&sh.low, (unsigned long long)low);
        } else {
            atomicMax((uint32_t*)&sh.high, (uint32_t)high);
            atomicMin((uint32_t*)&sh.low, (uint32_t)low);
        }
        __syncthreads();
        high = sh.high;
        low = sh.low;
        uint32_t n;
        do {
            const int shift = max(bits_of(high - low) - 11, 0); // kBins parts
            clear(sh.sub.count, sh.sub.mass);
            sweep_some(test, [&](T l, uint32_t) {
                const Key k = key_of(l);
                if (k >= low && k <= high) {
                    const uint32_t s = (uint32_t)((high - k) >> shift);
                    atomicAdd(&sh.sub.count[s], 1u);
                    atomicAdd(&sh.sub.mass[s], mass_of(weight(l)));
                }
            });
            __syncthreads();
            running_sums(sh.sub.count, sh.sub.mass);
            const uint32_t s = first_bin(sh.sub.count, sh.sub.mass, [&](uint32_t c, unsigned long long m) {
                return done(count + c, mass + m);
            });
            n = sh.sub.count[s] - (s ? sh.sub.count[s - 1] : 0);
            if (s) {
                count += sh.sub.count[s - 1];
                mass += sh.sub.mass[s - 1];
            }
            high -= (Key)s << shift;
            const Key span = ((Key)1 << shift) - 1;
            low = high - low > span ? high - span : low;
            __syncthreads();
        } while (n > kList && low < high);
        g.keyed = true;
        g.low = low;
        g.high = high;
        return n;
    }

    // Index of the nth word (from 1, in ascending order) of this value.
    __device__ __forceinline__ uint32_t nth_of_value(T value, uint32_t nth) {
        uint32_t seen = 0;
        if (tid == 0)
            sh.found = 0xffffffffu;
        __syncthreads();
        if (nth == 1) {
            sweep_some([&](T l) { return l == value; }, [&](T, uint32_t i) { atomicMin(&sh.found, i); });
            __syncthreads();
            return sh.found;
        }
        for (int64_t i0 = 0; i0 < vocab; i0 += kThreads) {
            const int64_t i = i0 + tid;
            const bool hit = i < vocab && logits[i] == value;
            const unsigned long long ballot = __ballot(hit);
            if ((tid & 63) == 0)
                sh.wave_count[tid >> 6] = (uint32_t)__popcll(ballot);
            __syncthreads();
            uint32_t before = seen, all = seen;
#pragma unroll
            for (int w = 0; w < kWaves; ++w) {
                before += w < tid >> 6 ? sh.wave_count[w] : 0;
                all += sh.wave_count[w];
            }
            if (hit && before + __builtin_amdgcn_mbcnt_hi((uint32_t)(ballot >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)ballot, 0)) + 1 == nth)
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

    // A row whose largest logit is infinite: the words that have it share all the mass. Which of them it is.
    __device__ __forceinline__ uint32_t among_infinite(T value, int64_t top_k, double top_p, double u) {
        if (tid == 0)
            sh.listed = 0;
        __syncthreads();
        sweep_some([&](T l) { return l == value; }, [&](T, uint32_t) { atomicAdd(&sh.listed, 1u); });
        __syncthreads();
        double n = (double)(top_k > 0 ? min(top_k, (int64_t)sh.listed) : (int64_t)sh.listed);
        if (top_p < 1.0)
            n = fmax(ceil(top_p * n), 1.0);
        u = u > 0.0 ? fmin(u, 1.0) : 0.0;
        return (uint32_t)fmin(floor(u * n) + 1.0, n);
    }
};

// What a row asks for, with entries outside their range held to it.
struct Settings {
    double temperature, top_p, min_p;
    int64_t top_k;
    bool greedy, weigh; // the largest logit; every word's weight is needed
    template <typename T>
    __device__ __forceinline__ Settings(const SampleParams<T>& p, int64_t row) {
        temperature = p.temperatures ? p.temperatures[row] : p.temperature;
        top_p = p.top_ps ? p.top_ps[row] : p.top_p;
        min_p = p.min_ps ? p.min_ps[row] : p.min_p;
        min_p = min_p > 0.0 ? fmin(min_p, 1.0) : 0.0;
        top_k = p.top_ks ? p.top_ks[row] : p.top_k;
        greedy = !(temperature > 0.0 && top_k != 1 && !(top_p <= 0.0));
        // a small top-k is cut by the lanes' maxima
        weigh = !(top_k > 0 && top_k <= kThreads / 2);
    }
};

// Adds the weights of the row's words to the bins of sh.mass, their numbers to those of sh.count when
// `counted`; returns this lane's part of the mass of those that weigh min_p or more. No branches, so that a
// pack's words go through the long chains side by side: what is out of reach adds nothing to the bin
// beyond the last.
template <typename T>
__device__ __forceinline__ unsigned long long weigh_words(const Row<T>& r, Shared<T>& sh, double min_p, bool counted) {
    unsigned long long own = 0;
    r.sweep([&](const auto& q, uint32_t) {
        constexpr int N = (int)(sizeof(q.v) / sizeof(T));
        int b[N];
        double w[N];
#pragma unroll
        for (int j = 0; j < N; ++j) {
            double rest;
            b[j] = r.bin_at(r.depth(q.v[j]), &rest);
            w[j] = r.weight_at(b[j], rest);
        }
#pragma unroll
        for (int j = 0; j < N; ++j)
            atomicAdd(&sh.mass[b[j]], r.mass_of(w[j]));
        if (min_p > 0.0)
#pragma unroll
            for (int j = 0; j < N; ++j)
                own += b[j] < kBins && w[j] >= min_p ? r.mass_of(w[j]) : 0;
        if (counted)
#pragma unroll
            for (int j = 0; j < N; ++j)
                atomicAdd(&sh.count[b[j]], 1u);
    });
    return own;
}

// The largest logit that the lanes hold, in all of them.
template <typename T>
__device__ __forceinline__ T group_max(T v, Shared<T>& sh) {
    v = wave_max(v);
    if ((threadIdx.x & 63) == 0)
        sh.wave_top[threadIdx.x >> 6] = v;
    __syncthreads();
    return row_max(sh.wave_top[threadIdx.x & 15]);
}
template <typename T>
__device__ __forceinline__ T own_max(const Row<T>& r) {
    T top = -std::numeric_limits<T>::infinity();
    r.sweep([&](const auto& q, uint32_t) {
#pragma unroll
        for (int j = 0; j < (int)(sizeof(q.v) / sizeof(T)); ++j)
            top = q.v[j] > top ? q.v[j] : top; // NaN: never
    });
    return top;
}

// A slice of a row: its largest logit; and zeros where the slices' weights will be added up.
template <typename T>
__global__ __launch_bounds__(kThreads) void slice_top_kernel(SampleParams<T> p) {
    __shared__ Shared<T> sh;
    const int tid = threadIdx.x;
    const int64_t row = blockIdx.y, first = blockIdx.x * p.slice;
    const Row<T> r{sh, p.logits + row * p.stride + first, std::min(p.slice, p.vocab - first), 0.0, 0.0, 0.0, tid, false};
    const T top = group_max(own_max(r), sh);
    if (tid == 0)
        p.tops[row * p.slices + blockIdx.x] = top;
    for (int b = blockIdx.x * kThreads + tid; b < kBins; b += p.slices * kThreads) {
        p.masses[row * kBins + b] = 0;
        p.counts[row * kBins + b] = 0;
    }
    if (blockIdx.x == 0 && tid == 0)
        p.above[row] = 0;
}

// A slice of a row: its words weighed, and what its bins hold added to the row's.
template <typename T>
__global__ __launch_bounds__(kThreads) void slice_weigh_kernel(SampleParams<T> p) {
    __shared__ Shared<T> sh;
    const int tid = threadIdx.x;
    const int64_t row = blockIdx.y, first = blockIdx.x * p.slice;
    const Settings q(p, row);
    T top = -std::numeric_limits<T>::infinity();
    for (int i = 0; i < p.slices; ++i)
        top = std::max(top, p.tops[row * p.slices + i]);
    if (q.greedy || !q.weigh || !(fabs((double)top) <= (double)std::numeric_limits<T>::max()))
        return; // the same for the whole workgroup
    Row<T> r{sh, p.logits + row * p.stride + first, std::min(p.slice, p.vocab - first), 0.0, 0.0, p.mass_scale, tid, true};
    r.fill_levels();
    r.set(top, q.temperature);
    r.clear(sh.count, sh.mass); // and a barrier behind the levels
    unsigned long long own = weigh_words(r, sh, q.min_p, q.top_k > 0);
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const int b = 2 * tid + j;
        if (sh.mass[b])
            atomicAdd(&p.masses[row * kBins + b], sh.mass[b]);
        if (sh.count[b])
            atomicAdd(&p.counts[row * kBins + b], sh.count[b]);
    }
    own = wave_sums(own);
    if ((tid & 63) == 63 && own)
        atomicAdd(&p.above[row], own);
}

template <typename T>
__global__ __launch_bounds__(kThreads) void sample_kernel(SampleParams<T> p) {
    typedef typename KeyOf<T>::type Key;
    __shared__ Shared<T> sh;
    const int tid = threadIdx.x;
    const int64_t row = p.first_row + blockIdx.x;
    Row<T> r{sh, p.logits + row * p.stride, p.vocab, 0.0, 0.0, p.mass_scale, tid, false};
    const Settings q(p, row);
    const double top_p = q.top_p, min_p = q.min_p;
    const int64_t top_k = q.top_k;
    const double u0 = p.u[row], u = u0 > 0.0 ? fmin(u0, 1.0) : 0.0;
    bool weigh = q.weigh;
    bool weighed = p.slices > 1 && weigh; // by the slices

    // the largest logit; each lane keeps its own
    const T none = -std::numeric_limits<T>::infinity();
    T own_top = none;
    if (weighed)
        own_top = tid < p.slices ? p.tops[row * p.slices + tid] : none;
    else
        own_top = own_max(r);
    const T top = group_max(own_top, sh);

    int32_t drawn = -1;        // every word is masked (or no number)
    T value = top;             // where a place among words of one value decides: the value, and which of
    uint32_t nth = 0;          // them, counted from 1
    if (top > none && q.greedy) {
        nth = 1;
    } else if (top > std::numeric_limits<T>::max()) {
        nth = r.among_infinite(top, top_k, top_p, u);
    } else if (top > none) {
        r.set(top, q.temperature);
        auto target_of = [&](unsigned long long kept) {
            return min((unsigned long long)(u * (double)kept), kept - 1);
        };
        const bool short_row = p.vocab <= kList; // a list takes all of it: no bins, no cut in front
        if (short_row)
            weigh = weighed = false;
        for (bool again = true; again;) {
            again = false;
            unsigned long long own = 0, total = 0;
            uint32_t by_k = kBins, by_p = kBins, by_min_p = kBins;
            Until until{Until::REACHED, (uint32_t)max(top_k, (int64_t)0), 0.0, 0};
            r.weighed = weigh;
            if (weigh)
                r.fill_levels();
            if (!short_row) {
                r.clear(sh.count, sh.mass);
                if (weighed) {
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const int b = 2 * tid + j;
                        sh.mass[b] = p.masses[row * kBins + b];
                        sh.count[b] = p.counts[row * kBins + b];
                    }
                    own = tid == 0 ? p.above[row] : 0;
                } else if (weigh) {
                    own = weigh_words(r, sh, min_p, top_k > 0);
                } else if (own_top > none) {
                    atomicAdd(&sh.count[r.bin_of(own_top)], 1u);
                }
                __syncthreads();
                if (weigh && !(top_k > 0)) {
                    // nobody counts: a bin's words weigh its level times e^(-1/128) or more, which
                    // tells how many they are nearly enough to decide whether a list takes them
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const int b = 2 * tid + j;
                        const double each = fmax(sh.level[b] * 0.992 * p.mass_scale, 1.0);
                        sh.count[b] = (uint32_t)fmin(ceil((double)sh.mass[b] / each), (double)p.vocab);
                    }
                }
                r.running_sums(sh.count, sh.mass);
                total = sh.mass[kBins - 1];
                until.reached = top_p * (double)total;
                if (top_k > 0 && top_k <= (int64_t)sh.count[kBins - 1]) {
                    until.kind = Until::COUNT;
                    by_k = r.first_bin(sh.count, sh.mass, until);
                    until.kind = Until::REACHED;
                }
                if (weigh && top_p < 1.0)
                    by_p = r.first_bin(sh.count, sh.mass, until);
            }
            auto count_of = [&](uint32_t b0, uint32_t b1) { return sh.count[b1] - (b0 ? sh.count[b0 - 1] : 0); };
            if (min_p > 0.0)
                by_min_p = (uint32_t)fmin(-log(min_p) * kBinsPerUnit + 1.0, (double)kBins); // one to spare
            uint32_t last = min(min(by_k, by_p), by_min_p); // last bin of a list of all that is kept
            // p of what top-k leaves needs all of that in the list
            if (top_p < 1.0 && (!weigh || (top_k > 0 && by_k != kBins)))
                last = by_k;
            last = min(last, (uint32_t)kBins - 1);
            if (weigh && min_p > 0.0) {
                // mass of the words that min-p keeps: the sum of `own` over the workgroup
                own = wave_sums(own);
                if ((tid & 63) == 63)
                    sh.wave_mass[tid >> 6] = own;
                __syncthreads();
                own = of_lane(row_sums(sh.wave_mass[tid & 15]), 15);
                __syncthreads();
            }

            // ALL: everything kept in one list. Otherwise the cuts one by one: by COUNT what top-k
            // leaves, by MASS what top-p does; DRAW the word. Where top-p's cut is known to a bin the
            // draw is known to a few: BOTH gathers the words of both.
            enum { ALL, BY_COUNT, BOTH, BY_MASS, DRAW } stage = ALL;
            unsigned long long most = total; // mass kept, as far as it is cut
            Range<Key> g;
            g.keyed = false;
            uint32_t base_count = 0;
            unsigned long long base_mass = 0;
            if (weigh && sh.count[last] > kList)
                stage = by_k != kBins ? BY_COUNT : BOTH;
            for (bool more = true; more;) {
                uint32_t n = kList + 1;
                if (!g.keyed) {
                    if (stage == ALL) {
                        g.b0 = 0;
                        g.b1 = g.b2 = last;
                        n = 0; // tried whatever the counts say: they may be those of the lanes' maxima
                    } else if (stage == BOTH) {
                        until.kind = Until::REACHED;
                        const uint32_t cut = top_p < 1.0 ? r.first_bin(sh.count, sh.mass, until) : kBins;
                        if (min_p > 0.0)
                            most = min(most, own);
                        if (cut == kBins || (cut ? sh.mass[cut - 1] : 0) >= most) {
                            stage = DRAW; // top-p takes nothing away
                            continue;
                        }
                        base_mass = cut ? sh.mass[cut - 1] : 0;
                        until.kind = Until::PASSED;
                        until.passed = target_of(max(base_mass, 1ull));
                        g.b0 = r.first_bin(sh.count, sh.mass, until);
                        until.passed = target_of(min(most, sh.mass[cut]));
                        g.b1 = r.first_bin(sh.count, sh.mass, until);
                        g.b2 = cut;
                        n = count_of(g.b0, g.b1) + count_of(cut, cut);
                    } else {
                        until.kind = stage == BY_COUNT ? Until::COUNT : stage == BY_MASS ? Until::REACHED : Until::PASSED;
                        until.passed = target_of(most);
                        g.b0 = g.b1 = g.b2 = r.first_bin(sh.count, sh.mass, until);
                        base_count = g.b2 ? sh.count[g.b2 - 1] : 0;
                        base_mass = g.b2 ? sh.mass[g.b2 - 1] : 0;
                        n = count_of(g.b2, g.b2);
                    }
                } else {
                    n = 0; // narrowed to what fits
                }
                if (n <= kList)
                    n = r.gather(g);
                unsigned long long at = 0; // running mass at the word looked for
                uint32_t index = 0;
                if (n > kList) {
                    if (stage == ALL) {
                        if (!weigh) { // a crowd at the cut: weigh every word
                            weigh = again = true;
                            break;
                        }
                        stage = by_k != kBins ? BY_COUNT : BOTH;
                        continue;
                    }
                    if (stage == BOTH) {
                        stage = BY_MASS;
                        continue;
                    }
                    n = r.narrow(g, until, base_count, base_mass);
                    if (n <= kList)
                        continue;
                    // words of one value: the place follows from their common mass
                    value = value_of(g.high);
                    const unsigned long long each = r.mass_of(r.weight(value));
                    uint32_t lo = 1, hi = n;
                    while (lo < hi) {
                        const uint32_t mid = lo + (hi - lo) / 2;
                        if (until(base_count + mid, base_mass + mid * each))
                            hi = mid;
                        else
                            lo = mid + 1;
                    }
                    at = base_mass + lo * each;
                    if (stage == DRAW)
                        nth = lo;
                } else if (stage == ALL) {
                    uint32_t cut = top_k > 0 ? (uint32_t)min((int64_t)n, top_k) : n;
                    if (top_p < 1.0) {
                        // without a top-k that cuts, the list may end before the last word that counts
                        const double want = top_p * (double)(weigh && by_k == kBins ? total : sh.list.mass[cut - 1]);
                        cut = min(cut, r.listed_before(n, [&](uint32_t i) { return (double)sh.list.mass[i] >= want; }) + 1);
                    }
                    if (min_p > 0.0)
                        cut = min(cut, r.listed_before(n, [&](uint32_t i) {
                            return !(r.weight(value_of(sh.list.key[i])) >= min_p);
                        }));
                    const unsigned long long target = target_of(sh.list.mass[cut - 1]);
                    const uint32_t i = r.listed_before(cut, [&](uint32_t j) { return sh.list.mass[j] > target; });
                    drawn = (int32_t)sh.list.index[min(i, cut - 1)];
                    break;
                } else if (stage == BOTH) {
                    // running masses of the row: whole bins stand in the list, with a gap behind b1
                    const uint32_t head = g.b1 >= g.b2 ? n : r.listed_before(n, [&](uint32_t i) {
                        return r.bin_of(value_of(sh.list.key[i])) > (int)g.b1;
                    });
                    const unsigned long long base = g.b0 ? sh.mass[g.b0 - 1] : 0;
                    const unsigned long long skipped = head < n ? base_mass - sh.list.mass[head - 1] : 0;
                    auto upto = [&](uint32_t i) { return sh.list.mass[i] + (i < head ? base : skipped); };
                    const uint32_t end = min(r.listed_before(n, [&](uint32_t i) { return (double)upto(i) >= until.reached; }), n - 1);
                    const unsigned long long target = target_of(min(most, upto(end)));
                    const uint32_t i = r.listed_before(n, [&](uint32_t j) { return upto(j) > target; });
                    drawn = (int32_t)sh.list.index[min(i, n - 1)];
                    break;
                } else {
                    const uint32_t i = min(r.listed_before(n, [&](uint32_t j) {
                        return until(base_count + j + 1, base_mass + sh.list.mass[j]);
                    }), n - 1);
                    at = base_mass + sh.list.mass[i];
                    index = sh.list.index[i];
                    __syncthreads();
                }
                // one cut further
                g.keyed = false;
                if (stage == BY_COUNT) {
                    most = at;
                    until.reached = top_p * (double)most;
                    stage = BOTH;
                } else if (stage == BY_MASS) {
                    most = min(most, at);
                    stage = DRAW;
                } else {
                    drawn = (int32_t)index;
                    more = false;
                }
            }
        }
    }
    __syncthreads();
    if (nth)
        drawn = (int32_t)r.nth_of_value(value, nth);
    if (tid == 0)
        p.out[row] = drawn;
}

// Slices per row and the workspace for what they leave: host arithmetic on the sizes and on what the
// settings can ask for.
struct Plan {
    int slices;
    int64_t slice, bytes;
};
Plan plan_of(const cnh_sample_tokens_args* a) {
    Plan q{1, a->vocab, 0};
    const bool weighs = (a->top_ks || a->top_k == 0 || a->top_k > kThreads / 2) && (a->temperatures || a->temperature > 0.0);
    // One workgroup reads and weighs a word a lane at a time: a slice of 8192 words takes it 3 us, about what
    // the two more launches cost.
    if (weighs && a->rows > 0)
        q.slices = (int)std::max<int64_t>(1, std::min<int64_t>({16, 256 / a->rows, a->vocab / 8192}));
    if (q.slices > 1) {
        q.slice = ((a->vocab + q.slices - 1) / q.slices + 3) / 4 * 4;
        q.bytes = a->rows * (kBins * 12 + 8 + q.slices * (int64_t)dtype_size(a->dtype));
    }
    return q;
}

template <typename T>
int run(const cnh_sample_tokens_args* a, const Plan& q, hipStream_t st) {
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
    p.slices = q.slices;
    p.slice = q.slice;
    p.masses = static_cast<unsigned long long*>(a->workspace);
    p.above = p.masses + p.rows * kBins;
    p.tops = reinterpret_cast<T*>(p.above + p.rows);
    p.counts = reinterpret_cast<uint32_t*>(p.tops + p.rows * p.slices);
    if (p.slices > 1) {
        const dim3 grid(p.slices, (unsigned)p.rows);
        slice_top_kernel<T><<<grid, kThreads, 0, st>>>(p);
        slice_weigh_kernel<T><<<grid, kThreads, 0, st>>>(p);
    }
    for (p.first_row = 0; p.first_row < p.rows; p.first_row += 1 << 20) // a grid takes fewer than 2^32 lanes
        sample_kernel<T><<<(unsigned)std::min<int64_t>(p.rows - p.first_row, 1 << 20), kThreads, 0, st>>>(p);
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
    if (int rc = check(a, "cnh_sample_tokens_workspace"))
        return rc;
    return plan_of(a).bytes;
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
    const Plan q = plan_of(a);
    const Extent ws{"workspace", a->workspace, q.bytes};
    CNH_CHECK(q.bytes == 0 || (a->workspace && a->workspace_bytes >= q.bytes), -2,
              "%s: a workspace of %lld bytes is needed, %lld given", call, (long long)q.bytes,
              (long long)(a->workspace ? a->workspace_bytes : 0));
    CNH_CHECK(q.bytes == 0 || aligned_to(a->workspace, 16), -2, "%s: the workspace is not aligned to 16 bytes", call);
    for (const Extent* e : {&out, &logits, &ks, &doubles[0], &doubles[1], &doubles[2], &doubles[3]})
        CNH_CHECK(!overlap(ws, *e), -2, "%s: the workspace overlaps %s", call, e->what);
    if (int rc = ensure_init())
        return rc;
    DeviceScope dev;
    if (int rc = dev.enter())
        return rc;
    return a->dtype == CNH_F32 ? run<float>(a, q, as_stream(s)) : run<double>(a, q, as_stream(s));
}
