// draw.hip — one action (or token) a row from logits and one given uniform
// number a row: temperature, top-k, top-p, min-p, and a mask of what is legal.
//
// With m the largest unmasked logit and z = (x - m) / T, a row's candidates
// weigh w = floor(exp(z) 2^40): whole numbers, whose sums are exact in any
// order, so the answer is the same however a row is split, batched or
// scheduled (the floor takes at most 2^-40 of the likeliest's weight from a
// candidate). Candidates are ranked by logit, ties to the lowest index, and
//
//   top-k  keeps the first k;
//   top-p  of those keeps the ones before which less than p of their mass lies;
//   min-p  of those keeps exp(z) >= min_p;
//
// and the answer is the first index at which the running sum of the kept
// weights passes floor(u S), S being the sum. Its log-probability is
// z - log(S 2^-40).
//
// Ranking needs no sort: "the first so many in rank" is a threshold key (the
// logit's bits in an order that sorts as an integer) and how many of the
// candidates that equal it are taken, lowest index first.

#include "recurrent.h"

namespace {

typedef unsigned long long u64;

struct DrawArgs {
    const void* logits;
    int64_t row;               // elements between rows
    const uint8_t* mask;       // nonzero = legal, or null
    int64_t mask_row;
    const float* uniform;
    const float *temperature, *top_p, *min_p;   // per row, or null: the value below
    const int32_t* top_k;
    float temperature1, top_p1, min_p1;
    int32_t top_k1;
    int64_t* token;
    float* logp;
    int32_t rows, vocab;
};

// An integer that orders as the number does; -0 equals 0.
__device__ inline uint32_t key_of(float x) {
    const uint32_t u = __float_as_uint(x + 0.0f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ inline float of_key(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }

__device__ inline float z_of(float x, float m, float inv_t) { return x == m ? 0.0f : (x - m) * inv_t; }
__device__ inline u64 weight(float e) { return (u64)(e * 1099511627776.0f); }

// floor(part total / 2^24) for part <= 2^24 and total < 2^58, and its ceiling
__device__ inline u64 share(uint32_t part, u64 total, bool up) {
    const u64 low = (u64)part * (uint32_t)total;
    return (u64)part * (total >> 32) * 256 + ((low + (up ? 0xffffffu : 0u)) >> 24);
}

// Sums over a wave by cross-lane moves: eight lanes' neighbours, then rows of
// 16, then the halves; the total is in lane 63.
template <int CTRL, int ROWS>
__device__ inline u64 moved(u64 v) {
    const int lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)v, CTRL, ROWS, 0xf, false);
    const int hi = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)(v >> 32), CTRL, ROWS, 0xf, false);
    return (u64)(uint32_t)hi << 32 | (uint32_t)lo;
}

// The running sum over the lanes up to and with this one.
__device__ inline u64 wave_scan(u64 v) {
    v += moved<0x111, 0xf>(v);   // from 1, 2, 4, 8 lanes below in the row of 16
    v += moved<0x112, 0xf>(v);
    v += moved<0x114, 0xf>(v);
    v += moved<0x118, 0xf>(v);
    v += moved<0x142, 0xa>(v);   // lane 15 of rows 0 and 2 into rows 1 and 3
    v += moved<0x143, 0xc>(v);   // lane 31 into the upper half
    return v;
}

__device__ inline u64 last_lane(u64 v) {
    const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)v, 63);
    const uint32_t hi = __builtin_amdgcn_readlane((int)(uint32_t)(v >> 32), 63);
    return (u64)hi << 32 | lo;
}
__device__ inline u64 wave_sum(u64 v) { return last_lane(wave_scan(v)); }

// A row's settings; threads of a row agree on them.
struct Settings {
    float inv_t, min_p;
    uint32_t p24;      // top-p in units of 2^-24
    int k;             // 0: all
    bool greedy, cut;  // cut: top-p is on
};

__device__ inline Settings settings_of(const DrawArgs& a, int row) {
    Settings s;
    const float t = a.temperature ? a.temperature[row] : a.temperature1;
    s.greedy = !(t > 0.0f);
    s.inv_t = fmaxf(1.0f / t, 1.17549435e-38f);   // not 0: an infinite temperature leaves -inf where it is
    s.k = a.top_k ? a.top_k[row] : a.top_k1;
    if (s.k < 0 || s.k >= a.vocab) s.k = 0;
    const float p = a.top_p ? a.top_p[row] : a.top_p1;
    s.cut = p < 1.0f;
    s.p24 = s.cut && p > 0.0f ? (uint32_t)(p * 16777216.0f) : 0;
    const float least = a.min_p ? a.min_p[row] : a.min_p1;
    s.min_p = least < 1.0f ? least : 1.0f;
    return s;
}

// The 24 bits of a uniform number; what lies outside [0, 1) goes to its end.
__device__ inline uint32_t chance_of(float u) {
    const float v = u * 16777216.0f;
    return v >= 16777215.0f ? 16777215u : v > 0.0f ? (uint32_t)v : 0u;
}

// What a wave holds of a row: lanes take V neighbours, waves whole stretches,
// so that (wave, turn, lane, neighbour) is the order of indices.
template <typename T>
struct Row {
    static constexpr int V = 16 / sizeof(T);
    const T* p;
    const uint8_t* mask;
    int vocab;

    __device__ Row(const DrawArgs& a, int row)
        : p((const T*)a.logits + row * a.row), mask(a.mask ? a.mask + row * a.mask_row : nullptr), vocab(a.vocab) {}

    static constexpr uint32_t kNone = std::is_same<T, float>::value      ? 0xff800000u
                                      : std::is_same<T, _Float16>::value ? 0xfc00fc00u
                                                                         : 0xff80ff80u;   // -inf, or two of them
    struct Vec {
        uint32_t u[4];
        __device__ __forceinline__ float operator[](int j) const {
            if constexpr (sizeof(T) == 4)
                return __uint_as_float(u[j]);
            else if constexpr (std::is_same<T, __bf16>::value)
                return __uint_as_float(j & 1 ? u[j / 2] & 0xffff0000u : u[j / 2] << 16);
            else
                return (float)__builtin_bit_cast(_Float16, (uint16_t)(u[j / 2] >> (j & 1) * 16));
        }
    };
    // V logits from index i on; what is masked or past the end is -inf. A
    // vector past the end is read as the row's last whole one and moved down,
    // so no lane reads element by element (which costs the registers of eight).
    __device__ __forceinline__ Vec load(int i) const {
        const int at = i + V <= vocab ? i : vocab - V;
        Vec v;
        __builtin_memcpy(v.u, p + at, sizeof v.u);
        if (mask) {
            uint32_t ok[V / 4];
            __builtin_memcpy(ok, mask + at, V);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const bool legal = ok[j / 4] >> (j % 4) * 8 & 0xff;
                if constexpr (sizeof(T) == 4) {
                    v.u[j] = legal ? v.u[j] : kNone;
                } else {
                    const uint32_t half = j & 1 ? 0xffff0000u : 0xffffu;
                    v.u[j / 2] = legal ? v.u[j / 2] : (v.u[j / 2] & ~half) | (kNone & half);
                }
            }
        }
        int down = i - at;   // elements
        if (down > 0) {
            if constexpr (sizeof(T) == 2) {
                if (down & 1) {
#pragma unroll
                    for (int q = 0; q < 4; ++q) v.u[q] = (q < 3 ? v.u[q + 1] : kNone) << 16 | v.u[q] >> 16;
                }
                down >>= 1;
            }
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                if (down > q) {
                    v.u[0] = v.u[1];
                    v.u[1] = v.u[2];
                    v.u[2] = v.u[3];
                    v.u[3] = kNone;
                }
            }
        }
        return v;
    }
    // The same of a row that may be shorter than a vector.
    __device__ __forceinline__ Vec load_short(int i) const {
        if (vocab >= V) return load(i);
        Vec v;
#pragma unroll
        for (int q = 0; q < 4; ++q) v.u[q] = kNone;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            if (i + j >= vocab || (mask && !mask[i + j])) continue;
            if constexpr (sizeof(T) == 4)
                v.u[j] = __builtin_bit_cast(uint32_t, p[i + j]);
            else
                v.u[j / 2] = (v.u[j / 2] & (j & 1 ? 0xffffu : 0xffff0000u)) |
                             (uint32_t)__builtin_bit_cast(uint16_t, p[i + j]) << (j & 1) * 16;
        }
        return v;
    }
};

// The threshold: candidates whose key is above it are kept, and the first
// `take` of those that equal it.
struct Cut {
    uint32_t key;
    u64 take;
};

__device__ inline void answer(const DrawArgs& a, int row, int64_t token, float logp) {
    a.token[row] = token;
    a.logp[row] = logp;
}

__device__ inline float logp_of(float z, u64 total) { return z - logf((float)total * 9.094947017729282e-13f); }

// The lowest bit that tells two keys of a type apart: below it a positive
// number's are all 0 and a negative one's all 1.
template <typename T> constexpr int kLowBit = 0;
template <> constexpr int kLowBit<_Float16> = 13;
template <> constexpr int kLowBit<__bf16> = 16;
template <typename T>
__device__ inline uint32_t whole_key(uint32_t k) {
    return k & 0x80000000u ? k : k | ((1u << kLowBit<T>) - 1);
}

// ---- small vocabularies: a wave a row ------------------------------------------
// All of a row's weights are in registers; the thresholds are searched bit by
// bit, counts by ballots. 2048 rows of 243: 5.0 us, a launch and a row's chain
// of operations; with top-k 8.8, with top-p 19 (32 sums over the wave).
template <typename T, int E>   // E: candidates a lane
__global__ __launch_bounds__(256) void draw_small(DrawArgs a) {
    constexpr int V = Row<T>::V, TURNS = E / V;
    const int row = blockIdx.x * 4 + threadIdx.x / 64, lane = threadIdx.x & 63;
    if (row >= a.rows) return;
    const Settings s = settings_of(a, row);
    const Row<T> r(a, row);
    float x[E];
    float m = -INFINITY;
    bool bad = false;
#pragma unroll
    for (int q = 0; q < TURNS; ++q) {
        const auto v = r.load_short((q * 64 + lane) * V);
#pragma unroll
        for (int j = 0; j < V; ++j) {
            x[q * V + j] = v[j];
            m = fmaxf(m, x[q * V + j]);
            bad |= x[q * V + j] != x[q * V + j];
        }
    }
#pragma unroll
    for (int d = 32; d > 0; d /= 2) m = fmaxf(m, __shfl_xor(m, d));
    if (__ballot(bad)) return answer(a, row, -1, NAN);   // every lane writes the same
    if (m == -INFINITY) return answer(a, row, -1, 0.0f);
    const float inv_t = s.greedy ? 1.0f : s.inv_t;
    uint32_t key[E];
    u64 w[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
        key[e] = key_of(x[e]);
        w[e] = weight(expf(z_of(x[e], m, inv_t)));
    }
    Cut cut = {0, ~0ull};
    if (s.greedy || s.k == 1) {
        cut = {key_of(m), 1};
    } else {
        auto count = [&](uint32_t t) {   // of keys that reach t; what lies past the end does not
            int n = 0;
#pragma unroll
            for (int e = 0; e < E; ++e) n += __popcll(__ballot(key[e] >= t));
            return n;
        };
        if (s.k > 0) {
            uint32_t k = 0;
            for (int bit = 31; bit >= kLowBit<T>; --bit)
                if (count(k | 1u << bit) >= s.k) k |= 1u << bit;
            k = whole_key<T>(k);
            cut = {k, (u64)(s.k - (k == 0xffffffffu ? 0 : count(k + 1)))};
        }
        if (s.cut) {
            const u64 tie = s.k > 0 ? weight(expf(z_of(of_key(cut.key), m, inv_t))) : 0;
            auto mass = [&](uint32_t t) {   // of the kept ones that reach t
                u64 v = 0;
                int ties = 0;
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    v += key[e] >= t && key[e] > cut.key ? w[e] : 0;
                    if (s.k > 0) ties += __popcll(__ballot(key[e] >= t && key[e] == cut.key));
                }
                return wave_sum(v) + ((u64)ties < cut.take ? (u64)ties : cut.take) * tie;
            };
            u64 bound = share(s.p24, mass(0), true);
            if (bound == 0) bound = 1;
            uint32_t k = 0;
            for (int bit = 31; bit >= kLowBit<T>; --bit)
                if (mass(k | 1u << bit) >= bound) k |= 1u << bit;
            k = whole_key<T>(k);
            const u64 above = k == 0xffffffffu ? 0 : mass(k + 1);
            const u64 each = weight(expf(z_of(of_key(k), m, inv_t)));   // not 0: the bound is reached here
            u64 n = (bound - above + each - 1) / each;
            if (s.k > 0 && k == cut.key && n > cut.take) n = cut.take;
            cut = {k, n};
        }
    }
    // what is kept, in the order of indices: first the ties' ranks, then the running sums
    u64 total = 0, left = cut.take, before[TURNS], upto[TURNS];
#pragma unroll
    for (int q = 0; q < TURNS; ++q) {
        int ties = 0, rank = 0, all = 0;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const uint64_t b = __ballot(key[q * V + j] == cut.key);
            rank += __popcll(b & ((1ull << lane) - 1));
            all += __popcll(b);
        }
        u64 sum = 0;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const int e = q * V + j;
            bool keep = key[e] > cut.key;
            if (key[e] == cut.key) keep = (u64)(rank + ties++) < left;
            if (!keep || !(expf(z_of(x[e], m, inv_t)) >= s.min_p)) w[e] = 0;
            sum += w[e];
        }
        left -= (u64)all < left ? (u64)all : left;
        upto[q] = wave_scan(sum);
        const u64 turn = last_lane(upto[q]);
        upto[q] += total;
        before[q] = upto[q] - sum;
        total += turn;
    }
    const u64 target = share(chance_of(a.uniform[row]), total, false);
#pragma unroll
    for (int q = 0; q < TURNS; ++q) {
        if (target < before[q] || target >= upto[q]) continue;
        u64 run = before[q];
        int at = 0;
        float xt = 0.0f;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            if (target >= run && target < run + w[q * V + j]) {
                at = j;
                xt = x[q * V + j];
            }
            run += w[q * V + j];
        }
        answer(a, row, (q * 64 + lane) * V + at, s.greedy ? 0.0f : logp_of(z_of(xt, m, inv_t), total));
    }
}

// ---- large vocabularies: a workgroup a row ----------------------------------------
// The thresholds come from histograms in LDS: candidates fall into bins by
// their distance from the largest, a scan over the bins from the top finds the
// one in which the count or the mass passes its bound, and within that bin the
// keys are ranked against each other (or, where there are too many of them,
// fall into bins by key until one bin holds a single key or few enough).
// Beyond kFar weights are zero, and a threshold there is none. Sums are of
// integers, so the order in which the LDS takes them does not matter.
//
// Most draws need a fraction of a row, and all that follows happens on a list
// of it, if it fits the LDS: with top-k the candidates down to where at least k
// of them lie, going by the largest of each of a few thousand groups, which the
// pass that finds the largest of all keeps; with top-p alone those down to the
// bin of the threshold; with min-p alone those above that.
//
// 256 rows of 131072 bf16, a row a CU: the largest alone 16 us (67 MB at 4.2
// TB/s), top-k 50 39, with top-p after it 46: the row once more through the
// caches, then barriers. Without top-k every weight counts, and some 35 vector
// instructions a logit bound it: no filter 58 us, top-p 106 (spread logits,
// where a third of the row is kept and nothing fits a list: 151). One row of
// 50001 with top-k and top-p: 29 us, a CU's loads and the barriers.
//
// A short list goes through the bins as well: its 256 keys ranked whole, and
// each adding up those before it, need fewer barriers but as many LDS reads one
// after another (2048 rows of 8000 bf16: top-k 50 30 -> 35 us, top-p 56 -> 78).
//
// A top-p threshold after a top-k one needs no list of what top-k left: its
// bound is a share of that mass, which is reached at or above the top-k key,
// and among the ties there no later than the last one taken.
constexpr int kList = 256, kGroups = 4;   // keys ranked against each other; maxima a thread keeps
constexpr float kNear = 8.0f, kFar = 28.0f;
enum { kRangeNear, kRangeFar, kRangeAll };   // what the bins spread over: up to kNear, from there to kFar, up to kFar

template <int THREADS>
struct Shared {
    static constexpr int kBins = THREADS * 4, kCandidates = THREADS * 4;
    u64 mass[kBins];
    uint32_t count[kBins];
    uint32_t list[kList];
    uint32_t key_of[kCandidates], index_of[kCandidates];
    u64 part[THREADS / 64], part2[THREADS / 64];
    u64 turn[THREADS];            // kept mass of each turn of each wave
    int ties[THREADS];            // and its candidates at the threshold
    uint32_t fill, lo, hi, bin, key, at;
    u64 above_count, above_mass, take, before, mass_kept;
};

// Keeps the compiler from working on a lane's candidates side by side, which
// spills registers; the other waves fill the gaps.
__device__ __forceinline__ void one_by_one() { __builtin_amdgcn_sched_barrier(0); }

template <typename T, int THREADS>
struct Block {
    static constexpr int kBins = Shared<THREADS>::kBins, kCandidates = Shared<THREADS>::kCandidates;
    static constexpr int V = Row<T>::V, WAVES = THREADS / 64, N = kBins / THREADS, kAhead = 4;
    const Row<T> r;
    Shared<THREADS>& sh;
    const Settings& s;
    const int lane, wave;
    int turns;              // of each wave
    float m, inv_t;
    int have = -1;          // the range whose bins are in LDS
    int listed = 0;         // candidates in the list, if the rest happens there

    __device__ __forceinline__ Block(const DrawArgs& a, int row, Shared<THREADS>& shared, const Settings& settings)
        : r(a, row), sh(shared), s(settings), lane(threadIdx.x & 63), wave(threadIdx.x / 64) {
        const int all = (a.vocab + 64 * V - 1) / (64 * V);
        turns = (all + WAVES - 1) / WAVES;
    }
    // Calls f(turn, logits) for the wave's turns in order, with all lanes; the next few turns' loads are in flight.
    template <class F>
    __device__ __forceinline__ void each(F f) const {
        // where the lane starts is worked out anew by every pass: kept, it and what follows from it would be held in
        // registers through all of them
        int start = (wave * turns * 64 + lane) * V;
        asm volatile("" : "+v"(start));
        auto index = [&](int turn) { return start + turn * 64 * V; };
        typename Row<T>::Vec ahead[kAhead];
#pragma unroll
        for (int q = 0; q < kAhead; ++q) ahead[q] = r.load(index(q));
#pragma unroll 1
        for (int t = 0; t < turns; ++t) {
            float x[V];
#pragma unroll
            for (int j = 0; j < V; ++j) x[j] = ahead[0][j];
#pragma unroll
            for (int q = 0; q + 1 < kAhead; ++q) ahead[q] = ahead[q + 1];
            ahead[kAhead - 1] = r.load(index(t + kAhead));
            f(t, x);
        }
    }
    // Calls f(logit) for every candidate, of the list if there is one, in any order.
    template <class F>
    __device__ __forceinline__ void candidates(F f) const {
        if (listed) {
            for (int i = threadIdx.x; i < listed; i += THREADS) f(of_key(sh.key_of[i]));
        } else {
            each([&](int, float(&x)[V]) {
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    one_by_one();
                    f(x[j]);
                }
            });
        }
    }
    __device__ __forceinline__ float z(float x) const { return z_of(x, m, inv_t); }
    __device__ __forceinline__ u64 w(float x) const { return weight(expf(z(x))); }

    __device__ __forceinline__ u64 sum(u64 v) const {
        v = wave_sum(v);
        __syncthreads();
        if (lane == 0) sh.part[wave] = v;
        __syncthreads();
        u64 t = 0;
#pragma unroll 2
        for (int j = 0; j < WAVES; ++j) t += sh.part[j];
        return t;
    }
    // The sum over the threads before this one, and over all.
    __device__ __forceinline__ u64 scan(u64 v, u64* all) const {
        const u64 u = wave_scan(v);
        const u64 t = last_lane(u);
        __syncthreads();
        if (lane == 0) sh.part[wave] = t;
        __syncthreads();
        u64 before = u - v, sum = 0;
#pragma unroll 2
        for (int j = 0; j < WAVES; ++j) {
            if (j < wave) before += sh.part[j];
            sum += sh.part[j];
        }
        *all = sum;
        return before;
    }

    // Empty bins, and an empty list.
    __device__ __forceinline__ void clear() {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < N; ++i) {
            sh.count[threadIdx.x + i * THREADS] = 0;
            if (s.cut) sh.mass[threadIdx.x + i * THREADS] = 0;
        }
        if (threadIdx.x == 0) sh.fill = 0, sh.lo = 0xffffffffu, sh.hi = 0;
        __syncthreads();
    }
    __device__ __forceinline__ void clear_list() {
        __syncthreads();
        if (threadIdx.x == 0) sh.fill = 0, sh.lo = 0xffffffffu, sh.hi = 0;
        __syncthreads();
    }
    // Distances (from, to] of a range, and its bins; -1: outside.
    __device__ __forceinline__ static int bin_of(float z, int range) {
        const float from = range == kRangeFar ? kNear : 0.0f, to = range == kRangeNear ? kNear : kFar;
        if (!(z > -to) || (range == kRangeFar && z > -from)) return -1;
        const int b = (int)((-z - from) * (kBins / (to - from)));
        return b < kBins ? b : kBins - 1;
    }
    // Fills the bins with a range: counts, for a threshold by count, and with
    // top-p masses.
    __device__ __forceinline__ void fill(int range, bool counts) {
        clear();
        candidates([&](float x) {
            const float zx = z(x);
            const int b = bin_of(zx, range);
            if (b >= 0) {
                if (counts) atomicAdd(&sh.count[b], 1u);
                if (s.cut) atomicAdd(&sh.mass[b], weight(expf(zx)));
            }
        });
        have = range;
        __syncthreads();
    }
    __device__ __forceinline__ void totals(u64* c, u64* v) const {
        u64 tc = 0, tv = 0;
#pragma unroll
        for (int i = 0; i < N; ++i) tc += sh.count[threadIdx.x + i * THREADS], tv += s.cut ? sh.mass[threadIdx.x + i * THREADS] : 0;
        *c = sum(tc);
        *v = sum(tv);
    }
    // The first bin at which the running count (or mass) reaches `bound`: into
    // sh.bin, with what lies in the bins before. False if none does.
    __device__ __forceinline__ bool find(bool by_mass, u64 bound) {
        u64 c[N], v[N], cs = 0, vs = 0;
        __syncthreads();
        if (threadIdx.x == 0) sh.bin = kBins;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            c[i] = sh.count[threadIdx.x * N + i];
            v[i] = s.cut ? sh.mass[threadIdx.x * N + i] : 0;
            cs += c[i];
            vs += v[i];
        }
        u64 all;
        u64 cb = scan(cs, &all), vb = s.cut ? scan(vs, &all) : 0;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const u64 before = by_mass ? vb : cb, n = by_mass ? v[i] : c[i];
            if (before < bound && before + n >= bound) {   // one thread's one bin
                sh.bin = threadIdx.x * N + i;
                sh.above_count = cb;
                sh.above_mass = vb;
            }
            cb += c[i];
            vb += v[i];
        }
        __syncthreads();
        return sh.bin < kBins;
    }
    // Keys of one bin, between lo and hi, into the list as far as they fit, and
    // their lowest and highest; how many there are.
    __device__ __forceinline__ uint32_t collect(int range, int bin, uint32_t lo, uint32_t hi) {
        clear_list();
        have = -1;
        candidates([&](float x) {
            if (bin_of(z(x), range) == bin) {
                const uint32_t k = key_of(x);
                if (k >= lo && k <= hi) {
                    const uint32_t at = atomicAdd(&sh.fill, 1u);
                    if (at < kList) sh.list[at] = k;
                    atomicMin(&sh.lo, k);
                    atomicMax(&sh.hi, k);
                }
            }
        });
        __syncthreads();
        return sh.fill;
    }
    // The threshold at which the running count or mass, from the top, reaches
    // `bound`; `kept`: the mass up to there (with top-p). False where it lies
    // among weights of zero.
    __device__ __forceinline__ bool threshold(bool by_mass, u64 bound, Cut* cut, u64* kept) {
        u64 above_c = 0, above_m = 0;
        int range = have;
        if (range < 0) fill(range = by_mass || listed ? kRangeAll : kRangeNear, !by_mass);
        if (!find(by_mass, bound)) {
            if (range != kRangeNear) return false;
            totals(&above_c, &above_m);
            fill(range = kRangeFar, !by_mass);
            if (!find(by_mass, bound - (by_mass ? above_m : above_c))) return false;
        }
        const int bin = (int)sh.bin;
        above_c += sh.above_count;
        above_m += sh.above_mass;
        uint32_t members = collect(range, bin, 0, 0xffffffffu);
        uint32_t lo = sh.lo, hi = sh.hi;
        while (members > kList && lo != hi) {
            int shift = 0;
            while ((hi - lo) >> shift >= (uint32_t)kBins) ++shift;
            clear();
            candidates([&](float x) {
                if (bin_of(z(x), range) == bin) {
                    const uint32_t k = key_of(x);
                    if (k >= lo && k <= hi) {
                        if (!by_mass) atomicAdd(&sh.count[(hi - k) >> shift], 1u);
                        if (s.cut) atomicAdd(&sh.mass[(hi - k) >> shift], w(x));
                    }
                }
            });
            find(by_mass, bound - (by_mass ? above_m : above_c));
            const uint32_t q = sh.bin;   // its keys: hi - k from q << shift on, 1 << shift of them
            above_c += sh.above_count;
            above_m += sh.above_mass;
            const uint32_t top = hi - (q << shift), width = (1u << shift) - 1;
            members = collect(range, bin, top - lo < width ? lo : top - width, top);
            lo = sh.lo;
            hi = sh.hi;
        }
        if (lo == hi) {
            if (threadIdx.x == 0) {
                const u64 v = w(of_key(lo));
                sh.key = lo;
                sh.take = by_mass ? (bound - above_m + v - 1) / v : bound - above_c;
                sh.mass_kept = above_m + sh.take * v;
            }
        } else if (threadIdx.x < members) {
            const uint32_t k = sh.list[threadIdx.x];
            u64 c = above_c, v = above_m, ties = 0;
#pragma unroll 2
            for (uint32_t i = 0; i < members; ++i) {
                const uint32_t o = sh.list[i];
                ties += o == k;
                if (o > k) {
                    c += 1;
                    if (s.cut) v += w(of_key(o));
                }
            }
            const u64 each_w = s.cut ? w(of_key(k)) : 0;
            const u64 before = by_mass ? v : c, all = by_mass ? ties * each_w : ties;
            if (before < bound && before + all >= bound) {   // ties write the same
                const u64 take = by_mass ? (bound - before + each_w - 1) / each_w : bound - before;
                sh.key = k;
                sh.take = take;
                sh.mass_kept = v + take * each_w;
            }
        }
        __syncthreads();
        *cut = {sh.key, sh.take};
        *kept = sh.mass_kept;
        return true;
    }
    // A logit that at least `want` candidates reach, going by the threads' group
    // maxima; false if none is found within kFar.
    __device__ __forceinline__ bool bound_of(const float (&group)[kGroups], int want, float* bound) {
        clear();
        have = -1;
#pragma unroll
        for (int q = 0; q < kGroups; ++q) {
            const int b = bin_of(z(group[q]), kRangeAll);
            if (b >= 0) atomicAdd(&sh.count[b], 1u);
        }
        if (!find(false, (u64)want)) return false;
        *bound = logit_below(sh.bin);
        return true;
    }
    // A logit no higher than those of a bin of kRangeAll. (A list may hold more
    // than it has to, so what is rounded off goes to be safe.)
    __device__ __forceinline__ float logit_below(uint32_t bin) const {
        return m - (float)(bin + 2) * (kFar / kBins) / inv_t;
    }
    // Lists the candidates that reach `bound`; false (and nothing listed) where
    // they do not fit or are fewer than `want`.
    __device__ __forceinline__ bool make_list(float bound, int want) {
        clear_list();
        have = -1;
        each([&](int t, float(&x)[V]) {
            int mine = 0;
#pragma unroll
            for (int j = 0; j < V; ++j) mine += x[j] >= bound;
            if (__ballot(mine != 0)) {
                const int upto = (int)wave_scan((u64)mine);
                int at = 0;
                if (lane == 63) at = (int)atomicAdd(&sh.fill, (uint32_t)upto);
                at = __builtin_amdgcn_readlane(at, 63) + upto - mine;
                const int i = ((wave * turns + t) * 64 + lane) * V;
#pragma unroll
                for (int j = 0; j < V; ++j)
                    if (x[j] >= bound) {
                        if (at < kCandidates) sh.key_of[at] = key_of(x[j]), sh.index_of[at] = (uint32_t)(i + j);
                        ++at;
                    }
            }
        });
        __syncthreads();
        const int n = (int)sh.fill;
        if (n > kCandidates || n < want) return false;
        listed = n;
        return true;
    }
};

template <typename T, int THREADS>
__global__ __launch_bounds__(THREADS) void draw_large(DrawArgs a) {
    typedef Block<T, THREADS> B;
    constexpr int V = B::V, WAVES = B::WAVES;
    __shared__ Shared<THREADS> sh;
    const int row = blockIdx.x;
    const Settings s = settings_of(a, row);
    B b(a, row, sh, s);

    // the largest, and whether anything is not a number
    float m = -INFINITY, group[kGroups];
    int first = 0;   // the turn in which this thread first met its largest
    bool bad = false;
#pragma unroll
    for (int q = 0; q < kGroups; ++q) group[q] = -INFINITY;
    b.each([&](int t, float(&x)[V]) {
        float top = x[0];
#pragma unroll
        for (int j = 0; j < V; ++j) {
            top = fmaxf(top, x[j]);
            bad |= x[j] != x[j];
        }
        if (top > m) {
            m = top;
            first = t;
        }
        group[0] = fmaxf(group[0], top);
        if ((t + 1) * kGroups / b.turns != t * kGroups / b.turns && t + 1 < b.turns) {   // on to the next group
#pragma unroll
            for (int q = kGroups - 1; q > 0; --q) group[q] = group[q - 1];
            group[0] = -INFINITY;
        }
    });
    const float mine_top = m;
#pragma unroll
    for (int d = 32; d > 0; d /= 2) m = fmaxf(m, __shfl_xor(m, d));
    const bool any_bad = __ballot(bad) != 0;
    if (b.lane == 0) sh.part[b.wave] = (u64)any_bad << 32 | __float_as_uint(m);
    __syncthreads();
    bad = false;
    for (int j = 0; j < WAVES; ++j) {
        bad |= sh.part[j] >> 32 != 0;
        m = fmaxf(m, __uint_as_float((uint32_t)sh.part[j]));
    }
    if (bad || m == -INFINITY) {   // nothing to draw from: no number among them, or nothing legal
        if (threadIdx.x == 0) answer(a, row, -1, bad ? NAN : 0.0f);
        return;
    }
    b.m = m;
    b.inv_t = s.greedy ? 1.0f : s.inv_t;

    if (s.greedy || s.k == 1) {   // the first of the largest
        if (threadIdx.x == 0) sh.lo = 0xffffffffu;
        __syncthreads();
        const uint32_t at = (uint32_t)((b.wave * b.turns + first) * 64 + b.lane);
        if (mine_top == m) atomicMin(&sh.lo, at);
        __syncthreads();
        if (mine_top == m && sh.lo == at) {
            const auto x = b.r.load((int)at * V);
            int j = V - 1;
#pragma unroll
            for (int q = V - 1; q >= 0; --q) j = x[q] == m ? q : j;
            answer(a, row, (int64_t)at * V + j, 0.0f);
        }
        return;
    }
    Cut cut = {0, ~0ull};
    {
        u64 kept = 0;
        bool of_k = false;
        float bound;
        constexpr int kMost = THREADS * kGroups / 2;   // half the groups: their maxima still tell
        if (s.k > 0) {
            if (s.k <= kMost && b.bound_of(group, s.k, &bound)) b.make_list(bound, s.k);
            of_k = b.threshold(false, (u64)s.k, &cut, &kept);
        }
        if (s.cut) {
            b.have = -1;
            if (!of_k) {   // a share of all there is
                b.listed = 0;
                b.fill(kRangeAll, false);
                u64 count;
                b.totals(&count, &kept);
            }
            u64 share_of = share(s.p24, kept, true);
            if (share_of == 0) share_of = 1;
            if (!of_k && b.find(true, share_of)) {
                // a list, if it has the promise to fit: a little over half the
                // groups reach that far
                bound = b.logit_below(sh.bin);
                u64 groups = 0;
#pragma unroll
                for (int q = 0; q < kGroups; ++q) groups += group[q] >= bound;
                if (b.sum(groups) <= THREADS * kGroups * 9 / 16) {
                    if (b.make_list(bound, 1)) {
                        // (rounding at logits of a million and more could leave some out)
                        u64 mass = 0;
                        b.candidates([&](float x) { mass += b.w(x); });
                        if (b.sum(mass) < share_of) b.listed = 0;
                    }
                }
            }
            b.threshold(true, share_of, &cut, &kept);
        } else if (!of_k && s.min_p > 0.0f) {
            b.listed = 0;
            // and a little more, if that is more than what is rounded off
            if (fabsf(m) * b.inv_t < 2e4f) b.make_list(m + (logf(s.min_p) - 0.01f) / b.inv_t, 1);
        }
    }

    const float tie_e = expf(b.z(of_key(cut.key)));
    const u64 tie = tie_e >= s.min_p ? weight(tie_e) : 0;
    sh.turn[threadIdx.x] = 0;
    sh.ties[threadIdx.x] = 0;
    __syncthreads();
    if (b.listed) {
        // all that is kept is in the list. Of the ties at the threshold the first
        // ones by index are: those after them leave it (with too many ties to
        // rank the row is gone through instead)
        u64 ties = 0;
        for (int i = threadIdx.x; i < b.listed; i += THREADS) ties += sh.key_of[i] == cut.key;
        ties = b.sum(ties);
        if (ties > cut.take && ties <= kList) {
            b.clear_list();
            for (int i = threadIdx.x; i < b.listed; i += THREADS)
                if (sh.key_of[i] == cut.key) sh.list[atomicAdd(&sh.fill, 1u)] = sh.index_of[i];
            __syncthreads();
            for (int i = threadIdx.x; i < b.listed; i += THREADS)
                if (sh.key_of[i] == cut.key) {
                    u64 rank = 0;
                    for (int q = 0; q < (int)ties; ++q) rank += sh.list[q] < sh.index_of[i];
                    if (rank >= cut.take) sh.key_of[i] = 0;   // below any threshold
                }
            ties = cut.take;
            __syncthreads();
        }
        // the kept mass of each stretch of indices, the stretch that holds the
        // answer, and in it the candidates
        int width = 0;   // bits of a stretch
        while ((a.vocab - 1) >> width >= THREADS) ++width;
        if (ties <= cut.take) {
            for (int i = threadIdx.x; i < b.listed; i += THREADS) {
                const uint32_t k = sh.key_of[i];
                if (k >= cut.key && k != 0) {
                    const float e = expf(b.z(of_key(k)));
                    if (e >= s.min_p) atomicAdd(&sh.turn[sh.index_of[i] >> width], weight(e));
                }
            }
            __syncthreads();
            const u64 mine = sh.turn[threadIdx.x];
            u64 total;
            const u64 before = b.scan(mine, &total);
            const u64 target = share(chance_of(a.uniform[row]), total, false);
            if (before <= target && target < before + mine) {   // one thread
                sh.at = threadIdx.x;
                sh.before = before;
                sh.fill = 0;
            }
            __syncthreads();
            const uint32_t at = sh.at;
            u64* kept_w = sh.mass;   // of the stretch's candidates, at most 256
            for (int i = threadIdx.x; i < b.listed; i += THREADS) {
                const uint32_t k = sh.key_of[i], x = sh.index_of[i];
                if (x >> width != at || k < cut.key || k == 0) continue;
                const float e = expf(b.z(of_key(k)));
                if (!(e >= s.min_p)) continue;
                const uint32_t q = atomicAdd(&sh.fill, 1u);
                sh.list[q] = x;
                sh.count[q] = k;
                kept_w[q] = weight(e);
            }
            __syncthreads();
            const int n = (int)sh.fill;
            if ((int)threadIdx.x >= n) return;
            const uint32_t x = sh.list[threadIdx.x];
            u64 run = sh.before;
            for (int i = 0; i < n; ++i)
                if (sh.list[i] < x) run += kept_w[i];
            if (run <= target && target < run + kept_w[threadIdx.x])
                answer(a, row, x, s.greedy ? 0.0f : logp_of(b.z(of_key(sh.count[threadIdx.x])), total));
            return;
        }
        sh.turn[threadIdx.x] = 0;
        __syncthreads();
    }

    // each turn's kept mass, and its candidates at the threshold
    b.each([&](int t, float(&x)[V]) {
        u64 sum = 0;
        int eq = 0;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            one_by_one();
            const uint32_t k = key_of(x[j]);
            if (k > cut.key) {
                const float e = expf(b.z(x[j]));
                if (e >= s.min_p) sum += weight(e);
            }
            eq += __popcll(__ballot(k == cut.key));
        }
        sum = __ballot(sum != 0) ? wave_sum(sum) : 0;
        if (b.lane == 0) {
            sh.turn[b.wave * b.turns + t] = sum;
            sh.ties[b.wave * b.turns + t] = eq;
        }
    });
    __syncthreads();
    const u64 eq = sh.ties[threadIdx.x];
    u64 total;
    const u64 ties_before = b.scan(eq, &total);
    u64 allowed = cut.take > ties_before ? cut.take - ties_before : 0;
    const u64 mine = sh.turn[threadIdx.x] + (eq < allowed ? eq : allowed) * tie;
    const u64 before = b.scan(mine, &total);
    u64 target = share(chance_of(a.uniform[row]), total, false);
    if (before <= target && target < before + mine) {   // one thread
        sh.at = threadIdx.x;
        sh.before = before;
        sh.take = allowed;
    }
    __syncthreads();
    if (b.wave != 0) return;
    // the turn that holds it, candidate by candidate
    const int i = ((int)sh.at * 64 + b.lane) * V;
    target -= sh.before;
    allowed = sh.take;
    const auto raw = b.r.load(i);
    float x[V];
#pragma unroll
    for (int j = 0; j < V; ++j) x[j] = raw[j];
    u64 w[V], sum = 0;
    int rank = 0, own = 0;
#pragma unroll
    for (int j = 0; j < V; ++j)
        rank += __popcll(__ballot(key_of(x[j]) == cut.key) & ((1ull << b.lane) - 1));
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const uint32_t k = key_of(x[j]);
        const float e = expf(b.z(x[j]));
        bool keep = k > cut.key;
        if (k == cut.key) keep = (u64)(rank + own++) < allowed;
        w[j] = keep && e >= s.min_p ? weight(e) : 0;
        sum += w[j];
    }
    u64 run = wave_scan(sum) - sum;
    if (target < run || target >= run + sum) return;
    int at = 0;
    float xt = 0.0f;
#pragma unroll
    for (int j = 0; j < V; ++j) {
        if (target >= run && target < run + w[j]) {
            at = j;
            xt = x[j];
        }
        run += w[j];
    }
    answer(a, row, i + at, s.greedy ? 0.0f : logp_of(b.z(xt), total));
}

}  // namespace

extern "C" {

SDFR_API int32_t sdfr_draw(const SdfrDraw* s, void* stream) {
    const char* fn = "sdfr_draw";
    g_rec_err[0] = '\0';
    if (!s) return rec_fail(-1, "%s: null descriptor", fn);
    if (s->rows < 0 || s->vocab < 1 || s->vocab > (1 << 18))
        return rec_fail(-2, "%s: rows must not be negative and the vocabulary 1 to %d (got %d and %d)", fn, 1 << 18,
                        s->rows, s->vocab);
    if (!rec_float(s->dtype)) return rec_fail(-3, "%s: dtype must be f32, f16 or bf16 (got %d)", fn, s->dtype);
    if (s->rows == 0) return 0;
    if (!s->logits || !s->uniform || !s->token || !s->logp) return rec_fail(-1, "%s: null pointer argument", fn);
    hipStream_t st = (hipStream_t)stream;
    DrawArgs a;
    a.logits = s->logits;
    a.row = s->logits_row;
    a.mask = s->mask;
    a.mask_row = s->mask_row;
    a.uniform = s->uniform;
    a.temperature = s->temperature;
    a.top_k = s->top_k;
    a.top_p = s->top_p;
    a.min_p = s->min_p;
    a.temperature1 = s->temperature1;
    a.top_k1 = s->top_k1;
    a.top_p1 = s->top_p1;
    a.min_p1 = s->min_p1;
    a.token = s->token;
    a.logp = s->logp;
    a.rows = s->rows;
    a.vocab = s->vocab;
    // Which kernel (bf16, no filter / top-k 50 / top-p 0.9 / both, us): a wave a
    // row up to 1024, what its registers hold: 2048 rows of 1000 8 / 11 / 19 / 28,
    // by a workgroup 20 / 24 / 33 / 32. Workgroups of 256 threads, several a CU,
    // up to 16384 (512 rows of 16000 23 / 20 / 41 / 23, 1024 threads 29 / 36 / 61 /
    // 50; one row of 20000 22 / 18 / 41 / 21 and 17 / 19 / 33 / 26), and up to
    // 65536, as far as a stretch's candidates fit kList, where there are more rows
    // than CUs (512 rows of 60000 63 / 37 / 115 / 40 and 68 / 53 / 122 / 66; 256
    // rows 53 / 33 / 100 / 36 and 33 / 26 / 61 / 32).
    rec_typed(s->dtype, [&](auto v) {
        typedef decltype(v) T;
        const unsigned small = (unsigned)((s->rows + 3) / 4);
        if (s->vocab <= 512)
            draw_small<T, 8><<<small, 256, 0, st>>>(a);
        else if (s->vocab <= 1024)
            draw_small<T, 16><<<small, 256, 0, st>>>(a);
        else if (s->vocab <= (s->rows > 256 ? 65536 : 16384))
            draw_large<T, 256><<<s->rows, 256, 0, st>>>(a);
        else
            draw_large<T, 1024><<<s->rows, 1024, 0, st>>>(a);
        return 0;
    });
    return rec_launched(fn);
}

}  // extern "C"
