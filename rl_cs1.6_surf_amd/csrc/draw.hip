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

__device__ inline u64 wave_sum(u64 v) {
#pragma unroll
    for (int m = 32; m > 0; m /= 2) v += __shfl_xor(v, m);
    return v;
}

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

// What a row's threads hold of it: lanes take V neighbours, waves whole
// stretches, so that (wave, turn, lane, neighbour) is the order of indices.
template <typename T, int THREADS>
struct Row {
    static constexpr int V = 16 / sizeof(T);
    static constexpr int WAVES = THREADS / 64;
    const T* p;
    const uint8_t* mask;
    int vocab, from, to, lane;

    __device__ Row(const DrawArgs& a, int row) {
        p = (const T*)a.logits + row * a.row;
        mask = a.mask ? a.mask + row * a.mask_row : nullptr;
        vocab = a.vocab;
        lane = threadIdx.x & 63;
        const int turn = 64 * V;
        const int turns = (vocab + turn - 1) / turn;
        const int each = (turns + WAVES - 1) / WAVES * turn;
        const int64_t f = (int64_t)(threadIdx.x / 64) * each;
        from = f < vocab ? (int)f : vocab;
        to = vocab - from < each ? vocab : from + each;
    }
    // V logits at index i; what is masked or past the end is -inf
    __device__ void load(int i, float (&x)[V]) const {
        if (i + V <= vocab) {
            T r[V];
            __builtin_memcpy(r, p + i, sizeof r);
#pragma unroll
            for (int j = 0; j < V; ++j) x[j] = (float)r[j];
            if (mask) {
                uint8_t ok[V];
                __builtin_memcpy(ok, mask + i, V);
#pragma unroll
                for (int j = 0; j < V; ++j)
                    if (!ok[j]) x[j] = -INFINITY;
            }
        } else {
#pragma unroll
            for (int j = 0; j < V; ++j) x[j] = i + j < vocab && (!mask || mask[i + j]) ? (float)p[i + j] : -INFINITY;
        }
    }
    // Calls f(first index, logits) for this lane's vectors, in order, by all lanes of the wave alike.
    template <class F>
    __device__ void each(F f) const {
        for (int i = from; i < to; i += 64 * V) {
            float x[V];
            load(i + lane * V, x);
            f(i + lane * V, x);
        }
    }
};

// Sums over the block of one or two numbers a thread.
template <int THREADS>
__device__ inline u64 block_sum(u64 v, u64* lds) {
    v = wave_sum(v);
    if constexpr (THREADS == 64) return v;
    __syncthreads();
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x / 64] = v;
    __syncthreads();
    u64 s = 0;
#pragma unroll
    for (int j = 0; j < THREADS / 64; ++j) s += lds[j];
    return s;
}

template <typename T, int THREADS>
__global__ __launch_bounds__(THREADS) void draw_rows(DrawArgs a) {
    constexpr int WAVES = THREADS / 64;
    __shared__ u64 lds[WAVES + 1];
    __shared__ u64 sums[WAVES];
    __shared__ int ties[WAVES];
    const int row = blockIdx.x;
    const int wave = threadIdx.x / 64;
    const Settings s = settings_of(a, row);
    const Row<T, THREADS> r(a, row);
    constexpr int V = Row<T, THREADS>::V;

    // the largest, and whether anything is not a number
    float m = -INFINITY;
    bool bad = false;
    r.each([&](int, float(&x)[V]) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
            m = fmaxf(m, x[j]);
            bad |= x[j] != x[j];
        }
    });
    uint32_t top = key_of(m);
#pragma unroll
    for (int k = 32; k > 0; k /= 2) {
        const uint32_t o = __shfl_xor(top, k);
        top = o > top ? o : top;
    }
    const bool any_bad = __ballot(bad) != 0;
    if (WAVES > 1) {
        if ((threadIdx.x & 63) == 0) lds[wave] = (u64)any_bad << 32 | top;
        __syncthreads();
        bad = false;
        for (int j = 0; j < WAVES; ++j) {
            bad |= lds[j] >> 32 != 0;
            top = (uint32_t)lds[j] > top ? (uint32_t)lds[j] : top;
        }
        __syncthreads();
    } else {
        bad = any_bad;
    }
    m = of_key(top);
    if (bad || m == -INFINITY) {   // nothing to draw from: no number among them, or nothing legal
        if (threadIdx.x == 0) {
            a.token[row] = -1;
            a.logp[row] = bad ? NAN : 0.0f;
        }
        return;
    }
    const float inv_t = s.greedy ? 1.0f : s.inv_t;

    // the threshold: candidates above `key` are kept, and the first `take` that equal it
    uint32_t key = 0;
    u64 take = ~0ull;
    if (s.greedy || s.k == 1) {
        key = top;
        take = 1;
    } else {
        u64 limit = ~0ull;   // of those at the top-k threshold
        uint32_t kkey = 0;
        if (s.k > 0) {       // the largest key that at least k candidates reach
            for (int bit = 31; bit >= 0; --bit) {
                const uint32_t t = kkey | 1u << bit;
                u64 n = 0;
                r.each([&](int i, float(&x)[V]) {
#pragma unroll
                    for (int j = 0; j < V; ++j) n += i + j < a.vocab && key_of(x[j]) >= t;
                });
                if (block_sum<THREADS>(n, lds) >= (u64)s.k) kkey = t;
            }
            u64 above = 0;
            r.each([&](int, float(&x)[V]) {
#pragma unroll
                for (int j = 0; j < V; ++j) above += key_of(x[j]) > kkey;
            });
            limit = s.k - block_sum<THREADS>(above, lds);
            key = kkey;
            take = limit;
        }
        if (s.cut) {
            // mass of the kept ones that reach t, ties at the top-k threshold counted as far as they are kept
            auto mass = [&](uint32_t t) {
                u64 w = 0, eq = 0;
                r.each([&](int, float(&x)[V]) {
#pragma unroll
                    for (int j = 0; j < V; ++j) {
                        const uint32_t k = key_of(x[j]);
                        if (k >= t && (k > kkey || s.k == 0)) w += weight(expf(z_of(x[j], m, inv_t)));
                        eq += s.k > 0 && k >= t && k == kkey;
                    }
                });
                w = block_sum<THREADS>(w, lds);
                if (s.k > 0) {
                    eq = block_sum<THREADS>(eq, lds);
                    w += (eq < limit ? eq : limit) * weight(expf(z_of(of_key(kkey), m, inv_t)));
                }
                return w;
            };
            u64 bound = share(s.p24, mass(0), true);
            if (bound == 0) bound = 1;
            uint32_t pkey = 0;   // the largest key whose mass reaches the bound
            for (int bit = 31; bit >= 0; --bit) {
                const uint32_t t = pkey | 1u << bit;
                if (mass(t) >= bound) pkey = t;
            }
            const u64 above = pkey == 0xffffffffu ? 0 : mass(pkey + 1);
            const u64 each = weight(expf(z_of(of_key(pkey), m, inv_t)));   // not 0: the bound is reached here
            u64 n = (bound - above + each - 1) / each;
            if (pkey == kkey && s.k > 0 && n > limit) n = limit;
            key = pkey;
            take = n;
        }
    }

    // each wave's kept mass and ties
    u64 w = 0;
    int eq = 0;
    r.each([&](int, float(&x)[V]) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const uint32_t k = key_of(x[j]);
            const float e = expf(z_of(x[j], m, inv_t));
            if (k > key && e >= s.min_p) w += weight(e);
            eq += k == key;
        }
    });
    w = wave_sum(w);
    eq = (int)wave_sum((u64)eq);
    const float tie_e = expf(z_of(of_key(key), m, inv_t));
    const u64 tie = tie_e >= s.min_p ? weight(tie_e) : 0;
    if ((threadIdx.x & 63) == 0) {
        sums[wave] = w;
        ties[wave] = eq;
    }
    __syncthreads();
    u64 total = 0, before = 0, left = take, allowed = 0;
    for (int j = 0; j < WAVES; ++j) {
        const u64 n = (u64)ties[j] < left ? (u64)ties[j] : left;
        if (j == wave) before = total, allowed = left;
        total += sums[j] + n * tie;
        left -= n;
    }
    u64 target = share(chance_of(a.uniform[row]), total, false);
    const u64 mine = w + ((u64)eq < allowed ? (u64)eq : allowed) * tie;
    if (target < before || target >= before + mine) return;
    // the wave that holds it walks its stretch
    target -= before;
    for (int i = r.from; i < r.to; i += 64 * V) {
        float x[V];
        u64 run[V], lane_sum = 0;
        r.load(i + r.lane * V, x);
        int lane_ties = 0;
#pragma unroll
        for (int j = 0; j < V; ++j) lane_ties += key_of(x[j]) == key;
        int ties_before = lane_ties;   // inclusive scan over the lanes
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
            const int o = __shfl_up(ties_before, d);
            if (r.lane >= d) ties_before += o;
        }
        const int turn_ties = __shfl(ties_before, 63);
        int rank = ties_before - lane_ties;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const uint32_t k = key_of(x[j]);
            const float e = expf(z_of(x[j], m, inv_t));
            bool keep = k > key;
            if (k == key) keep = (u64)rank++ < allowed;
            if (keep && e >= s.min_p) lane_sum += weight(e);
            run[j] = lane_sum;
        }
        u64 upto = lane_sum;
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
            const u64 o = __shfl_up(upto, d);
            if (r.lane >= d) upto += o;
        }
        const u64 turn_sum = __shfl(upto, 63);
        if (target < turn_sum) {
            const u64 lo = upto - lane_sum;
            if (target >= lo && target < upto) {
                int j = 0;
                while (run[j] + lo <= target) ++j;
                a.token[row] = i + r.lane * V + j;
                float xj = x[0];
#pragma unroll
                for (int q = 1; q < V; ++q)
                    if (q == j) xj = x[q];
                a.logp[row] = s.greedy ? 0.0f
                                       : z_of(xj, m, inv_t) - logf((float)total * 9.094947017729282e-13f);
            }
            return;
        }
        target -= turn_sum;
        allowed -= (u64)turn_ties < allowed ? (u64)turn_ties : allowed;
    }
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
    rec_typed(s->dtype, [&](auto v) {
        typedef decltype(v) T;
        if (s->vocab <= 1024)
            draw_rows<T, 64><<<s->rows, 64, 0, st>>>(a);
        else if (s->vocab <= 8192)
            draw_rows<T, 256><<<s->rows, 256, 0, st>>>(a);
        else
            draw_rows<T, 1024><<<s->rows, 1024, 0, st>>>(a);
        return 0;
    });
    return rec_launched(fn);
}

}  // extern "C"
