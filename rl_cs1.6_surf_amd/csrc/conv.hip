// conv.hip — the short causal convolution of a policy's memory: each channel's
// last `width` inputs, weighted, plus a bias, through SiLU or not; its
// gradients; and, as the call of length 1, its step for a single token.
//
//   pre[t] = bias + sum_j w[width-1-j] x[t-j],  j = 0 .. width-1
//   y[t]   = pre sigmoid(pre), or pre
//
// x before the first step comes from `state` (the last width-1 inputs of the
// call before, oldest first; zeros without one). Where a sequence begins
// (resets) nothing from before it is seen. Backwards, with dpre the gradient
// of pre:
//
//   dx[t] = sum_j w[width-1-j] dpre[t+j]     (j that see t)
//   dw[width-1-j] = sum_t dpre[t] x[t-j],    dbias = sum_t dpre[t]
//
// A thread takes 16 bytes of channels of one sequence and walks a run of
// steps with the window in registers, so inputs are read once but for the
// run's first width-1 rows.

#include "recurrent.h"

namespace {

using namespace rec;

constexpr int kRun = 16;       // steps a thread walks
constexpr int kMaxWidth = 8;

struct ConvArgs {
    const void* x;
    int64_t x_b, x_t;
    const float *weight, *bias;   // (channels, width), (channels) or null
    const uint8_t* resets;
    int64_t resets_b, resets_t;
    const void* state;            // (batch, width-1, channels) or null
    void* y;
    int64_t y_b, y_t;
    void* state_out;              // dense, or null
    int64_t length;
    int batch, channels, width, silu;
    int vecs, runs;               // channel vectors a row, runs a sequence
};

struct ConvGradArgs {
    const void* dy;
    int64_t dy_b, dy_t;
    const void* dstate_out;       // dense like state, or null
    void* dx;                     // dense (batch, length, channels)
    void* dstate;                 // dense like state, or null
    float* sums;                  // (partial rows, width + 1, channels)
    int rows;                     // partial rows
    int64_t jobs;                 // batch * runs
};

// V channels of a row. Rows of odd sizes or strides start anywhere: the loads
// go by bytes (global memory takes any address), and a row's last vector by
// elements.
template <typename T, int V>
__device__ inline void load_row(const T* p, int n, float (&v)[V]) {
    if (n >= V) {
        T r[V];
        __builtin_memcpy(r, p, sizeof r);
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = (float)r[i];
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = i < n ? (float)p[i] : 0.0f;
    }
}

template <typename T, int V>
__device__ inline void store_row(T* p, int n, const float (&v)[V]) {
    if (n >= V) {
        T r[V];
#pragma unroll
        for (int i = 0; i < V; ++i) r[i] = (T)v[i];
        __builtin_memcpy(p, r, sizeof r);
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (i < n) p[i] = (T)v[i];
    }
}

// Row t of the input, t >= -(width-1): before the first step, of the state.
template <typename T, int V>
__device__ inline void load_input(const ConvArgs& a, int b, int64_t t, int c, int n, float (&v)[V]) {
    if (t >= 0) {
        load_row<T, V>((const T*)a.x + b * a.x_b + t * a.x_t + c, n, v);
    } else if (a.state && t >= -(int64_t)(a.width - 1)) {
        load_row<T, V>((const T*)a.state + ((int64_t)b * (a.width - 1) + (a.width - 1 + t)) * a.channels + c, n, v);
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = 0.0f;
    }
}

__device__ inline bool begins(const ConvArgs& a, int b, int64_t t) {
    return a.resets && t >= 0 && t < a.length && a.resets[b * a.resets_b + t * a.resets_t] != 0;
}

// How many of the steps before t the window at t sees: up to width - 1, fewer
// where a sequence begins in between.
__device__ inline int sight_at(const ConvArgs& a, int b, int64_t t) {
    int s = 0;
    while (s < a.width - 1 && !begins(a, b, t - s)) ++s;
    return s;
}

__device__ inline int next_sight(const ConvArgs& a, int b, int64_t t, int sight) {
    return begins(a, b, t) ? 0 : sight < a.width - 1 ? sight + 1 : a.width - 1;
}

template <int V>
__device__ inline void shift_in(float (&win)[V], const float (&v)[V]) {
#pragma unroll
    for (int i = 0; i < V; ++i) win[i] = v[i];
}

template <int W, int V>
__device__ inline void load_weights(const ConvArgs& a, int c, int n, float (&w)[W][V], float (&bias)[V]) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
        bias[i] = i < n && a.bias ? a.bias[c + i] : 0.0f;
#pragma unroll
        for (int j = 0; j < W; ++j)   // w[j]: the weight of the input j steps back
            w[j][i] = i < n && j < a.width ? a.weight[(int64_t)(c + i) * a.width + a.width - 1 - j] : 0.0f;
    }
}

// pre at a step whose window is win[0] (now) .. win[W-1]; the first `sight`
// steps back are seen. What is not seen is not multiplied: it may be anything.
template <int W, int V>
__device__ inline void convolve(const float (&win)[W][V], const float (&w)[W][V], const float (&bias)[V], int sight,
                                float (&pre)[V]) {
#pragma unroll
    for (int i = 0; i < V; ++i) pre[i] = __builtin_fmaf(w[0][i], win[0][i], bias[i]);
#pragma unroll
    for (int j = 1; j < W; ++j)
        if (j <= sight) {
#pragma unroll
            for (int i = 0; i < V; ++i) pre[i] = __builtin_fmaf(w[j][i], win[j][i], pre[i]);
        }
}

template <typename T, int W, int V>
__global__ __launch_bounds__(256) void conv_forward(ConvArgs a) {
    const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int64_t job = id / a.vecs;
    if (job >= (int64_t)a.batch * a.runs) return;
    const int c = (int)(id % a.vecs) * V, n = a.channels - c;
    const int b = (int)(job / a.runs);
    const int64_t t0 = job % a.runs * kRun;
    const int64_t t1 = t0 + kRun < a.length ? t0 + kRun : a.length;
    float w[W][V], bias[V], win[W][V];
    load_weights<W, V>(a, c, n, w, bias);
#pragma unroll
    for (int j = 1; j < W; ++j) load_input<T, V>(a, b, t0 - j, c, n, win[j - 1]);   // shifted at the first step
    int sight = a.resets ? sight_at(a, b, t0 - 1) : a.width - 1;
    T* yp = (T*)a.y + b * a.y_b + c;
    for (int64_t t = t0; t < t1; ++t) {
#pragma unroll
        for (int j = W - 1; j > 0; --j) shift_in<V>(win[j], win[j - 1]);
        load_input<T, V>(a, b, t, c, n, win[0]);
        sight = next_sight(a, b, t, sight);
        float pre[V];
        convolve<W, V>(win, w, bias, sight, pre);
        if (a.silu) {
#pragma unroll
            for (int i = 0; i < V; ++i) pre[i] *= sigmoid(pre[i]);
        }
        store_row<T, V>(yp + t * a.y_t, n, pre);
    }
    if (a.state_out && t1 == a.length) {
        // the window the next call starts from; what it must not see is cleared
        const float none[V] = {};
        T* so = (T*)a.state_out + (int64_t)b * (a.width - 1) * a.channels + c;
#pragma unroll
        for (int j = 0; j < W - 1; ++j)
            if (j < a.width - 1)
                store_row<T, V>(so + (int64_t)(a.width - 2 - j) * a.channels, n, j <= sight ? win[j] : none);
    }
}

// A thread walks the runs of its share one after another with its sums of dw
// and dbias in registers. Within a run it goes W - 1 steps past the end, whose
// dpre the run's last inputs get their gradients from.
template <typename T, int W, int V>
__global__ __launch_bounds__(256) void conv_backward(ConvArgs a, ConvGradArgs g) {
    const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int64_t share = id / a.vecs;
    if (share >= g.rows) return;
    const int c = (int)(id % a.vecs) * V, n = a.channels - c;
    float w[W][V], bias[V], dw[W][V], db[V];
    load_weights<W, V>(a, c, n, w, bias);
#pragma unroll
    for (int i = 0; i < V; ++i) {
        db[i] = 0.0f;
#pragma unroll
        for (int j = 0; j < W; ++j) dw[j][i] = 0.0f;
    }
    for (int64_t job = share; job < g.jobs; job += g.rows) {
        const int b = (int)(job / a.runs);
        const int64_t t0 = job % a.runs * kRun;
        const int64_t t1 = t0 + kRun < a.length ? t0 + kRun : a.length;
        // steps t0 .. end-1 have a dpre; the run owns the gradients of inputs
        // t0 .. t1-1, the first one those of the state too
        const int64_t end = t1 + W - 1 < a.length ? t1 + W - 1 : a.length;
        float win[W][V], acc[W][V];   // acc[j]: gradient of the input j steps back, so far
#pragma unroll
        for (int j = 1; j < W; ++j) load_input<T, V>(a, b, t0 - j, c, n, win[j - 1]);
#pragma unroll
        for (int j = 0; j < W; ++j)
#pragma unroll
            for (int i = 0; i < V; ++i) acc[j][i] = 0.0f;
        int sight = a.resets ? sight_at(a, b, t0 - 1) : a.width - 1;
        const T* dyp = (const T*)g.dy + b * g.dy_b + c;
        auto put = [&](int64_t t, float (&v)[V]) {   // the gradient of input t is whole
            if (t >= t0 && t < t1) {
                store_row<T, V>((T*)g.dx + ((int64_t)b * a.length + t) * a.channels + c, n, v);
            } else if (t0 == 0 && t < 0 && g.dstate && t >= -(int64_t)(a.width - 1)) {
                store_row<T, V>((T*)g.dstate + ((int64_t)b * (a.width - 1) + a.width - 1 + t) * a.channels + c, n, v);
            }
        };
        for (int64_t t = t0; t < end; ++t) {
#pragma unroll
            for (int j = W - 1; j > 0; --j) {
                shift_in<V>(win[j], win[j - 1]);
                shift_in<V>(acc[j], acc[j - 1]);
            }
#pragma unroll
            for (int i = 0; i < V; ++i) acc[0][i] = 0.0f;
            load_input<T, V>(a, b, t, c, n, win[0]);
            sight = next_sight(a, b, t, sight);
            float d[V];
            load_row<T, V>(dyp + t * g.dy_t, n, d);
            if (a.silu) {
                float pre[V];
                convolve<W, V>(win, w, bias, sight, pre);
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const float s = sigmoid(pre[i]);
                    d[i] *= s * __builtin_fmaf(pre[i], 1.0f - s, 1.0f);
                }
            }
            const bool own = t < t1;
#pragma unroll
            for (int j = 0; j < W; ++j)
                if (j <= sight) {
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        acc[j][i] = __builtin_fmaf(w[j][i], d[i], acc[j][i]);
                        if (own) dw[j][i] = __builtin_fmaf(d[i], win[j][i], dw[j][i]);
                    }
                }
            if (own) {
#pragma unroll
                for (int i = 0; i < V; ++i) db[i] += d[i];
            }
            put(t - (W - 1), acc[W - 1]);
        }
        // inputs whose later readers lie past the sequence's end; the window
        // handed on holds the last ones
#pragma unroll
        for (int j = W - 2; j >= 0; --j) {
            const int64_t t = end - 1 - j;
            if (end == a.length && g.dstate_out && j < a.width - 1 && j <= sight) {
                float v[V];
                load_row<T, V>((const T*)g.dstate_out + ((int64_t)b * (a.width - 1) + a.width - 2 - j) * a.channels + c,
                               n, v);
#pragma unroll
                for (int i = 0; i < V; ++i) acc[j][i] += v[i];
            }
            if (end == a.length) put(t, acc[j]);
        }
    }
    float* s = g.sums + share * (a.width + 1) * a.channels + c;
#pragma unroll
    for (int j = 0; j < W; ++j)
        if (j < a.width) {
#pragma unroll
            for (int i = 0; i < V; ++i)
                if (i < n) s[(int64_t)j * a.channels + i] = dw[j][i];
        }
#pragma unroll
    for (int i = 0; i < V; ++i)
        if (i < n) s[(int64_t)a.width * a.channels + i] = db[i];
}

// dw and dbias from the shares' sums, always in the same order.
__global__ __launch_bounds__(1024) void conv_sums(const float* __restrict__ sums, float* dw, float* dbias, int rows,
                                                  int width, int channels) {
    __shared__ float lds[16][64];
    const int64_t cols = (int64_t)(width + 1) * channels;
    const int64_t c = (int64_t)blockIdx.x * 64 + threadIdx.x;
    float s = 0.0f;
    if (c < cols)
        for (int64_t r = threadIdx.y; r < rows; r += 16) s += sums[r * cols + c];
    lds[threadIdx.y][threadIdx.x] = s;
    __syncthreads();
    if (threadIdx.y != 0 || c >= cols) return;
    for (int j = 1; j < 16; ++j) s += lds[j][threadIdx.x];
    const int j = (int)(c / channels), d = (int)(c % channels);
    if (j < width)
        dw[(int64_t)d * width + width - 1 - j] = s;
    else if (dbias)
        dbias[d] = s;
}

int vec_of(int32_t dtype) { return dtype == SDFR_F32 ? 4 : 8; }

int32_t check_conv(const char* fn, const SdfrConv* s) {
    g_rec_err[0] = '\0';
    if (!s) return rec_fail(-1, "%s: null descriptor", fn);
    if (s->batch < 0 || s->length < 0 || s->channels < 1)
        return rec_fail(-2, "%s: bad sizes (batch %d, length %lld, channels %d)", fn, s->batch, (long long)s->length,
                        s->channels);
    if (s->width < 1 || s->width > kMaxWidth)
        return rec_fail(-2, "%s: width must be 1 to %d (got %d)", fn, kMaxWidth, s->width);
    if (!rec_float(s->dtype)) return rec_fail(-3, "%s: dtype must be f32, f16 or bf16 (got %d)", fn, s->dtype);
    const int64_t runs = (s->length + kRun - 1) / kRun, vecs = (s->channels + vec_of(s->dtype) - 1) / vec_of(s->dtype);
    if (s->channels > (1 << 24) || runs > 0x3fffffff || s->batch * runs > ((int64_t)1 << 38) / vecs)
        return rec_fail(-2, "%s: sizes too large", fn);
    if (!s->weight) return rec_fail(-1, "%s: null weight", fn);
    if (s->batch > 0 && s->length > 0 && (!s->x || !s->y)) return rec_fail(-1, "%s: null pointer argument", fn);
    if (s->length > kRun && s->state && s->state == s->state_out)
        return rec_fail(-2, "%s: the state is updated in place in calls of up to %d steps only", fn, kRun);
    return 0;
}

ConvArgs conv_args(const SdfrConv* s) {
    ConvArgs a;
    a.x = s->x;
    a.x_b = s->x_b;
    a.x_t = s->x_t;
    a.weight = s->weight;
    a.bias = s->bias;
    a.resets = s->resets;
    a.resets_b = s->resets_b;
    a.resets_t = s->resets_t;
    a.state = s->width > 1 ? s->state : nullptr;
    a.y = s->y;
    a.y_b = s->y_b;
    a.y_t = s->y_t;
    a.state_out = s->width > 1 ? s->state_out : nullptr;
    a.length = s->length;
    a.batch = s->batch;
    a.channels = s->channels;
    a.width = s->width;
    a.silu = s->silu;
    a.vecs = (s->channels + vec_of(s->dtype) - 1) / vec_of(s->dtype);
    a.runs = (int)((s->length + kRun - 1) / kRun);
    return a;
}

// Partial sums the gradients of the parameters are gathered in: enough shares
// to fill the machine, few enough that their sum is cheap.
int conv_rows(const ConvArgs& a) {
    const int64_t jobs = (int64_t)a.batch * a.runs;
    const int64_t rows = (256 * 1024 + a.vecs - 1) / a.vecs;
    return (int)(jobs < rows ? jobs : rows);
}

template <class F>
int32_t with_width(int width, F f) {
    if (width <= 4) return f(std::integral_constant<int, 4>());
    return f(std::integral_constant<int, 8>());
}

}  // namespace

extern "C" {

SDFR_API int32_t sdfr_conv(const SdfrConv* s, void* stream) {
    const char* fn = "sdfr_conv";
    int32_t rc = check_conv(fn, s);
    if (rc) return rc;
    if (s->batch == 0) return 0;
    if (s->length == 0) return rec_fail(-2, "%s: length must be positive", fn);
    hipStream_t st = (hipStream_t)stream;
    const ConvArgs a = conv_args(s);
    const unsigned blocks = (unsigned)(((int64_t)a.batch * a.runs * a.vecs + 255) / 256);
    rec_typed(s->dtype, [&](auto v) {
        typedef decltype(v) T;
        return with_width(s->width, [&](auto w) {
            conv_forward<T, decltype(w)::value, 16 / sizeof(T)><<<blocks, 256, 0, st>>>(a);
            return 0;
        });
    });
    return rec_launched(fn);
}

SDFR_API int64_t sdfr_conv_grad_workspace_bytes(const SdfrConv* s) {
    const int32_t rc = check_conv("sdfr_conv_grad_workspace_bytes", s);
    if (rc) return rc;
    const ConvArgs a = conv_args(s);
    return (int64_t)conv_rows(a) * (s->width + 1) * s->channels * 4;
}

SDFR_API int32_t sdfr_conv_grad(const SdfrConv* s, const SdfrConvGrad* g, void* workspace, int64_t workspace_size,
                                void* stream) {
    const char* fn = "sdfr_conv_grad";
    int32_t rc = check_conv(fn, s);
    if (rc) return rc;
    if (!g) return rec_fail(-1, "%s: null gradient descriptor", fn);
    if (s->batch == 0 || s->length == 0) return rec_fail(-2, "%s: nothing to differentiate", fn);
    if (!g->dy || !g->dx || !g->dweight) return rec_fail(-1, "%s: null pointer argument", fn);
    const ConvArgs a = conv_args(s);
    const int64_t need = (int64_t)conv_rows(a) * (s->width + 1) * s->channels * 4;
    if (!workspace) return rec_fail(-1, "%s: null workspace", fn);
    if (workspace_size < need)
        return rec_fail(-2, "%s: workspace of %lld bytes needed (got %lld)", fn, (long long)need,
                        (long long)workspace_size);
    if ((uintptr_t)workspace & 63) return rec_fail(-2, "%s: workspace must be 64-byte aligned", fn);
    hipStream_t st = (hipStream_t)stream;
    ConvGradArgs ga;
    ga.dy = g->dy;
    ga.dy_b = g->dy_b;
    ga.dy_t = g->dy_t;
    ga.dstate_out = s->width > 1 ? g->dstate_out : nullptr;
    ga.dx = g->dx;
    ga.dstate = s->width > 1 ? g->dstate : nullptr;
    ga.sums = (float*)workspace;
    ga.rows = conv_rows(a);
    ga.jobs = (int64_t)a.batch * a.runs;
    const unsigned blocks = (unsigned)(((int64_t)ga.rows * a.vecs + 255) / 256);
    rec_typed(s->dtype, [&](auto v) {
        typedef decltype(v) T;
        return with_width(s->width, [&](auto w) {
            conv_backward<T, decltype(w)::value, 16 / sizeof(T)><<<blocks, 256, 0, st>>>(a, ga);
            return 0;
        });
    });
    conv_sums<<<(unsigned)(((int64_t)(s->width + 1) * s->channels + 63) / 64), dim3(64, 16), 0, st>>>(
        ga.sums, g->dweight, g->dbias, ga.rows, s->width, s->channels);
    return rec_launched(fn);
}

}  // extern "C"
