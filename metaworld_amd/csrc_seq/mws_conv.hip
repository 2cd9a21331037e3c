// mws_conv.hip -- the short causal convolution over tokens with its activation: forward, backward, one token.
//
//   s_t = b + sum_j w_j x_{t-K+1+j}, y_t = s_t sigmoid(s_t); ds_t = dy_t silu'(s_t)
//   dx_p = sum_j w_j ds_{p+K-1-j}, dw_j = sum_t ds_t x_{t-K+1+j}, db = sum_t ds_t
//
// where x of a token before the row's first comes from the state, and of one before the episode's first is zero.
//
// Bound by memory, 512 x 128 x 1024 bf16 forward in 55 us (4.9 TB/s; a copy of 4 GiB reaches 4.8), backward in 93 us (4.3 TB/s, the vector
// unit at it for most of the time), one token of 4096 x 1024 bf16 in 13 us (5.1 TB/s; of 4096 x 1023, one value to a lane, 14 us).  A lane keeps V neighbouring channels (one 16-byte access a token), a wave walks over a tile of tokens with the
// last K of them in registers, so that every value is read once but for K - 1 tokens at a tile's edge (backward 2 K - 2).  The episodes' beginnings
// of a tile are one 64-bit mask in scalar registers.
#include "mws_common.hpp"

namespace mws {

struct ConvArgs {
    const void *x, *weight, *bias, *state, *dy, *dlast;
    const uint8_t *reset;
    const int32_t *lengths;
    void *y, *last, *dx, *dstate;
    float *part;                 // [blocks over tiles][K + 1][width]
    int64_t batch, length, tiles;
    int64_t x_batch, x_time, dy_batch, dy_time, reset_batch, reset_time;
    int width, tile;             // tokens of one wave's walk
    bool wide;
};

constexpr int kMostTile = 32;    // a tile with the tokens around it that matter to it fits one 64-bit mask

__device__ __forceinline__ int64_t row_length(const int32_t *lengths, int64_t b, int64_t length) {
    if (lengths == nullptr) return length;
    int64_t n = lengths[b];
    return n < 0 ? 0 : n > length ? length : n;
}

// bit i: an episode begins at token from + i (i < count, tokens within [0, end))
__device__ __forceinline__ uint64_t reset_mask(const uint8_t *reset, int64_t at, int64_t stride, int64_t from, int count, int64_t end) {
    if (reset == nullptr) return 0;
    int lane = threadIdx.x % kWave;
    int64_t t = from + lane;
    return __ballot(lane < count && t >= 0 && t < end && reset[at + t * stride] != 0);
}

template <class T, int V> struct Chan {
    float v[V];
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int i = 0; i < V; i++) v[i] = 0;
    }
    __device__ __forceinline__ void set(const Vec<T, V> &r) {
#pragma unroll
        for (int i = 0; i < V; i++) v[i] = up<T>(r.v[i]);
    }
    __device__ __forceinline__ Vec<T, V> rounded() const {
        Vec<T, V> r;
#pragma unroll
        for (int i = 0; i < V; i++) r.v[i] = down<T>(v[i]);
        return r;
    }
};

// a lane's V x K weights lie next to each other
template <class T, int V, int K> __device__ __forceinline__ void taps(const ConvArgs &a, int e, Chan<T, V> (&w)[K], Chan<T, V> &b) {
    if (a.wide) {
        Vec<F32, V * K> r = load<F32, V * K>((const float *)a.weight + (int64_t)e * K);
#pragma unroll
        for (int i = 0; i < V * K; i++) w[i % K].v[i / K] = r.v[i];
    } else {
        Vec<T, V * K> r = load<T, V * K>((const typename T::raw *)a.weight + (int64_t)e * K);
#pragma unroll
        for (int i = 0; i < V * K; i++) w[i % K].v[i / K] = up<T>(r.v[i]);
    }
    if (a.bias == nullptr) b.zero();
    else if (a.wide) {
        Vec<F32, V> r = load<F32, V>((const float *)a.bias + e);
#pragma unroll
        for (int i = 0; i < V; i++) b.v[i] = r.v[i];
    } else b.set(load<T, V>((const typename T::raw *)a.bias + e));
}

// the input at token p of row b (p >= -(K - 1); below zero: the state)
template <class T, int V, int K> __device__ __forceinline__ Vec<T, V> input(const ConvArgs &a, int64_t b, int64_t p, int e) {
    using raw = typename T::raw;
    if (p >= 0) return load<T, V>((const raw *)a.x + b * a.x_batch + p * a.x_time + e);
    if (a.state != nullptr) return load<T, V>((const raw *)a.state + (b * (K - 1) + p + K - 1) * a.width + e);
    Vec<T, V> r;
#pragma unroll
    for (int i = 0; i < V; i++) r.v[i] = 0;
    return r;
}

// A lane's channels.  Where the width is no multiple of V the last lane steps back to V whole ones: it makes some values a second time,
// the same ones, and every access stays whole.  (Not where the state is updated in place.)
template <int V> struct Mine {
    int e;
    bool on;
    __device__ __forceinline__ Mine(int lane_of_row, int width) : e(lane_of_row * V), on(e < width) { e = e + V <= width ? e : width - V; }
};

template <class T, int V, int K> __global__ __launch_bounds__(256) void conv_forward(ConvArgs a) {
    using raw = typename T::raw;
    const Mine<V> m(blockIdx.y * kWave + threadIdx.x % kWave, a.width);
    int64_t item = (int64_t)blockIdx.x * (blockDim.x / kWave) + uniform(threadIdx.x / kWave);
    if (item >= a.batch * a.tiles) return;
    int64_t b = item / a.tiles, t0 = (item % a.tiles) * a.tile, t1 = t0 + a.tile < a.length ? t0 + a.tile : a.length;
    int64_t end = row_length(a.lengths, b, a.length), stop = t1 < end ? t1 : end;
    Chan<T, V> w[K], bias, x[K];
    taps<T, V, K>(a, m.e, w, bias);
    raw *y = (raw *)a.y + (b * a.length + t0) * a.width + m.e;
    // bit i: token t0 - (K - 1) + i
    uint64_t begins = reset_mask(a.reset, b * a.reset_batch, a.reset_time, t0 - (K - 1), a.tile + K - 1, end);
    int count = (int)(stop > t0 ? stop - t0 : 0);
    if (count > 0) {
        x[0].zero();
#pragma unroll
        for (int j = 1; j < K; j++) {
            x[j].set(input<T, V, K>(a, b, t0 - K + j, m.e));
            if (begins >> (j - 1) & 1)
#pragma unroll
                for (int i = 0; i < j; i++) x[i].zero();
        }
        begins >>= K - 1;
        const raw *from = (const raw *)a.x + b * a.x_batch + t0 * a.x_time + m.e;
        auto token = [&](const Vec<T, V> &in, bool first) __attribute__((always_inline)) {
#pragma unroll
            for (int j = 0; j + 1 < K; j++) x[j] = x[j + 1];
            if (first)
#pragma unroll
                for (int j = 0; j + 1 < K; j++) x[j].zero();
            x[K - 1].set(in);
            Chan<T, V> s = bias;
#pragma unroll
            for (int i = 0; i < V; i++) {
#pragma unroll
                for (int j = 0; j < K; j++) s.v[i] += w[j].v[i] * x[j].v[i];
                s.v[i] *= sigmoid_(s.v[i]);
            }
            if (m.on) store<T, V>(y, s.rounded());
            y += a.width;
        };
        // four tokens at a time, the next four under way meanwhile
        Vec<T, V> next[4];
        int i = 0;
        if (count >= 4) {
#pragma unroll
            for (int q = 0; q < 4; q++) next[q] = load<T, V>(from + q * a.x_time);
            for (; i + 4 <= count; i += 4) {
                Vec<T, V> in[4];
#pragma unroll
                for (int q = 0; q < 4; q++) in[q] = next[q];
                from += 4 * a.x_time;
                if (i + 8 <= count)
#pragma unroll
                    for (int q = 0; q < 4; q++) next[q] = load<T, V>(from + q * a.x_time);
#pragma unroll
                for (int q = 0; q < 4; q++) token(in[q], begins >> q & 1);
                begins >>= 4;
            }
        }
        for (; i < count; i++) {
            token(load<T, V>(from), begins & 1);
            from += a.x_time, begins >>= 1;
        }
    }
    Vec<T, V> none;
#pragma unroll
    for (int i = 0; i < V; i++) none.v[i] = 0;
    y = (raw *)a.y + b * a.length * a.width + m.e;
    for (int64_t t = t0 > end ? t0 : end; t < t1; t++)
        if (m.on) store<T, V>(y + t * a.width, none);
    // the state after the last token: the inputs of its episode among the last K - 1, by the tile that holds this token
    if (a.last != nullptr && t0 == (end > 0 ? (end - 1) / a.tile : 0) * a.tile) {
        uint64_t tail = reset_mask(a.reset, b * a.reset_batch, a.reset_time, end - (K - 1), K - 1, end);
#pragma unroll
        for (int j = 0; j + 1 < K; j++) {
            bool seen = (tail >> (j + 1)) == 0;          // none begins after token end - (K - 1) + j
            Vec<T, V> r = seen ? input<T, V, K>(a, b, end - (K - 1) + j, m.e) : none;
            if (m.on) store<T, V>((raw *)a.last + (b * (K - 1) + j) * a.width + m.e, r);
        }
    }
}

// A wave walks from its tile's first token to K - 1 tokens past it: it takes dw and db of its own tokens, and dx of them, whose last
// terms come from the tokens past the tile.  The state's K - 1 inputs count as tokens before the first.  Four waves to a SIMD: with the
// next four tokens under way they do not fit (12 x 1000 x 640 fp32 with the forward pass 41 us when it was built, 79 us so; with three waves 51 us).
template <class T, int V, int K> __global__ __launch_bounds__(256, 4) void conv_backward(ConvArgs a) {
    using raw = typename T::raw;
    int lane = threadIdx.x % kWave, wave = uniform(threadIdx.x / kWave), waves = blockDim.x / kWave;
    const Mine<V> m(blockIdx.y * kWave + lane, a.width);
    const bool put_dx = m.on && a.dx != nullptr, put_state = m.on && a.dstate != nullptr;
    Chan<T, V> w[K], bias, dw[K], db;
    taps<T, V, K>(a, m.e, w, bias);
#pragma unroll
    for (int j = 0; j < K; j++) dw[j].zero();
    db.zero();
    for (int64_t item = (int64_t)blockIdx.x * waves + wave; item < a.batch * a.tiles; item += (int64_t)gridDim.x * waves) {
        int64_t b = item / a.tiles, t0 = (item % a.tiles) * a.tile, t1 = t0 + a.tile < a.length ? t0 + a.tile : a.length;
        int64_t end = row_length(a.lengths, b, a.length), stop = t1 + K - 1 < end ? t1 + K - 1 : end, own = t1 < end ? t1 : end;
        uint64_t begins = reset_mask(a.reset, b * a.reset_batch, a.reset_time, t0 - (K - 1), a.tile + 2 * (K - 1), end);
        Chan<T, V> x[K], pend[K];
        x[0].zero();
#pragma unroll
        for (int j = 0; j < K; j++) pend[j].zero();
        int age = K;                                     // tokens since the episode's first, K at most
        raw *dx = (raw *)a.dx + (b * a.length + t0) * a.width + m.e, *dstate = (raw *)a.dstate + b * (K - 1) * a.width + m.e;
        int count = (int)(stop > t0 ? stop - t0 : 0), mine = (int)(own > t0 ? own - t0 : 0);
        if (count > 0) {
#pragma unroll
            for (int j = 1; j < K; j++) {
                x[j].set(input<T, V, K>(a, b, t0 - K + j, m.e));
                if (begins >> (j - 1) & 1) {
                    age = K - 1 - j;
#pragma unroll
                    for (int i = 0; i < j; i++) x[i].zero();
                }
            }
            begins >>= K - 1;
            const raw *dyp = (const raw *)a.dy + b * a.dy_batch + t0 * a.dy_time + m.e, *xp = (const raw *)a.x + b * a.x_batch + t0 * a.x_time + m.e;
            auto token = [&](const Vec<T, V> &in, const Vec<T, V> &out, bool first, bool here, int p) __attribute__((always_inline)) {
#pragma unroll
                for (int j = 0; j + 1 < K; j++) x[j] = x[j + 1];
                age = age < K ? age + 1 : K;
                if (first) {
                    age = 0;
#pragma unroll
                    for (int j = 0; j + 1 < K; j++) x[j].zero();
                }
                x[K - 1].set(in);
                Chan<T, V> s = bias, d;
                d.set(out);
#pragma unroll
                for (int i = 0; i < V; i++) {
#pragma unroll
                    for (int j = 0; j < K; j++) s.v[i] += w[j].v[i] * x[j].v[i];
                    float sig = sigmoid_(s.v[i]);
                    d.v[i] *= sig * (1.0f + s.v[i] * (1.0f - sig));
                }
#pragma unroll
                for (int j = 0; j + 1 < K; j++)
                    if (age >= K - 1 || K - 1 - j <= age)
#pragma unroll
                        for (int i = 0; i < V; i++) pend[j].v[i] += w[j].v[i] * d.v[i];
#pragma unroll
                for (int i = 0; i < V; i++) pend[K - 1].v[i] = w[K - 1].v[i] * d.v[i];
                if (here)
#pragma unroll
                    for (int i = 0; i < V; i++) {
                        db.v[i] += d.v[i];
#pragma unroll
                        for (int j = 0; j < K; j++) dw[j].v[i] += d.v[i] * x[j].v[i];
                    }
                // added up here: the compiler would put the sums off to where they are next asked for and keep their terms instead
#pragma unroll
                for (int i = 0; i < V; i++) {
                    asm volatile("" : "+v"(db.v[i]));
#pragma unroll
                    for (int j = 0; j < K; j++) asm volatile("" : "+v"(dw[j].v[i]), "+v"(pend[j].v[i]));
                }
                // token p has its last term (it is not among the row's last K - 1, which the state that the row leaves reaches)
                if (p >= 0) {
                    if (put_dx) store<T, V>(dx + (int64_t)p * a.width, pend[0].rounded());
                } else if (t0 == 0 && put_state) store<T, V>(dstate + (int64_t)(p + K - 1) * a.width, pend[0].rounded());
#pragma unroll
                for (int j = 0; j + 1 < K; j++) pend[j] = pend[j + 1];
            };
            int i = 0;
            for (; i + 4 <= mine; i += 4) {
                Vec<T, V> in[4], out[4];
#pragma unroll
                for (int q = 0; q < 4; q++) in[q] = load<T, V>(xp + q * a.x_time), out[q] = load<T, V>(dyp + q * a.dy_time);
#pragma unroll
                for (int q = 0; q < 4; q++) token(in[q], out[q], begins >> q & 1, true, i + q - (K - 1));
                begins >>= 4, xp += 4 * a.x_time, dyp += 4 * a.dy_time;
            }
            for (; i < count; i++) {
                token(load<T, V>(xp), load<T, V>(dyp), begins & 1, i < mine, i - (K - 1));
                begins >>= 1, xp += a.x_time, dyp += a.dy_time;
            }
        }
        // the K - 1 tokens before the end of the walk, where that is the row's: past the tile they are another wave's
        if (t0 + count == end && (count > 0 || t0 == 0)) {
            uint64_t tail = reset_mask(a.reset, b * a.reset_batch, a.reset_time, end - (K - 1), K - 1, end);
#pragma unroll
            for (int j = 0; j + 1 < K; j++) {
                int p = count - (K - 1) + j;
                if (t0 + p >= t1 || (p < 0 && t0 > 0)) continue;
                if (a.dlast != nullptr && (tail >> (j + 1)) == 0) {
                    Chan<T, V> d;
                    d.set(load<T, V>((const raw *)a.dlast + (b * (K - 1) + j) * a.width + m.e));
#pragma unroll
                    for (int i = 0; i < V; i++) pend[j].v[i] += d.v[i];
                }
                if (p >= 0) {
                    if (put_dx) store<T, V>(dx + (int64_t)p * a.width, pend[j].rounded());
                } else if (put_state) store<T, V>(dstate + (int64_t)(p + K - 1) * a.width, pend[j].rounded());
            }
        }
        Chan<T, V> none;
        none.zero();
        if (put_dx)
            for (int64_t t = t0 > end ? t0 : end; t < t1; t++) store<T, V>(dx + (t - t0) * a.width, none.rounded());
    }
    if (a.part == nullptr) return;
    // the block's sums: its waves' meet in shared memory, behind one barrier for all of them
    __shared__ float meet[4][(K + 1) * V][kWave];
    float *part = a.part + (int64_t)blockIdx.x * (K + 1) * a.width;
#pragma unroll
    for (int j = 0; j <= K; j++)
#pragma unroll
        for (int i = 0; i < V; i++) meet[wave][j * V + i][lane] = j < K ? dw[j < K ? j : 0].v[i] : db.v[i];
    __syncthreads();
    if (m.on)
        for (int r = wave; r < (K + 1) * V; r += waves) {
            float s = 0;
            for (int k = 0; k < waves; k++) s += meet[k][r][lane];
            part[(int64_t)(r / V) * a.width + m.e + r % V] = s;
        }
}

// One token: the window is the state and x; every value of the state is read and written once.  A lane keeps its channels' weights
// for up to kStepRows rows; a row is under way while the one before is worked on.
constexpr int kStepRows = 8;
template <class T, int V, int K> __global__ __launch_bounds__(256) void conv_step(ConvArgs a, int64_t groups, int64_t each) {
    using raw = typename T::raw;
    int64_t at = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (at >= each * groups) return;
    const int e = (int)(at % groups) * V;                 // V divides the width
    int64_t b0 = at / groups;                             // rows b0, b0 + each, ..
    Chan<T, V> w[K], bias;
    taps<T, V, K>(a, e, w, bias);
    Vec<T, V> next[K];
    bool next_first = false;
    auto fetch = [&](int64_t b) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < K; j++) next[j] = input<T, V, K>(a, b, j - (K - 1), e);
        next_first = a.reset != nullptr && a.reset[b * a.reset_batch] != 0;
    };
    fetch(b0);
    for (int64_t b = b0; b < a.batch; b += each) {
        Vec<T, V> in[K];
        bool first = next_first;
#pragma unroll
        for (int j = 0; j < K; j++) in[j] = next[j];
        if (b + each < a.batch) fetch(b + each);
        Chan<T, V> s = bias;
#pragma unroll
        for (int j = 0; j < K; j++)
#pragma unroll
            for (int i = 0; i < V; i++) {
                if (first && j + 1 < K) in[j].v[i] = 0;
                s.v[i] += w[j].v[i] * up<T>(in[j].v[i]);
            }
#pragma unroll
        for (int i = 0; i < V; i++) s.v[i] *= sigmoid_(s.v[i]);
        store<T, V>((raw *)a.y + b * a.width + e, s.rounded());
#pragma unroll
        for (int j = 0; j + 1 < K; j++) store<T, V>((raw *)a.last + (b * (K - 1) + j) * a.width + e, in[j + 1]);
    }
}

struct ConvOut {
    void *dweight, *dbias;
    int width, taps, type;
    bool wide;
    __device__ void operator()(int64_t col, float v) const {
        int j = (int)(col / width), e = (int)(col % width);
        void *to = j < taps ? dweight : dbias;
        int64_t at = j < taps ? (int64_t)e * taps + j : e;
        if (to == nullptr) return;
        if (wide || type == MWS_F32) ((float *)to)[at] = v;
        else if (type == MWS_BF16) ((uint16_t *)to)[at] = down<BF16>(v);
        else ((uint16_t *)to)[at] = down<F16>(v);
    }
};

// Channels of a lane: one 16-byte access, or one value where the row is narrower than that (or, where the state is updated in place,
// no multiple of it).  A tile of 32 tokens re-reads K - 1 of its neighbour's; where that leaves less than four waves to a SIMD, tiles
// get shorter.
static int conv_v(const mws_conv_args *a) {
    int v = a->type == MWS_F32 ? 4 : 8;
    return a->width >= v ? v : 1;
}
// backward four of any type: with eight the weights, inputs, sums and gradients of the taps leave two waves to a SIMD (512 x 128 x 1024
// bf16 with eight 118 us when with four it was 102 us)
static int conv_back_v(const mws_conv_args *a) { return a->width >= 4 ? 4 : 1; }
static int conv_tile(const mws_conv_args *a) {
    int64_t across = a->batch * ceil_div(a->width, kWave * conv_v(a));
    int tile = kMostTile;
    while (tile > 8 && across * ceil_div(a->length, tile) < 4 * kSimds) tile /= 2;
    return tile;
}
static int64_t conv_tiles(const mws_conv_args *a) { return a->length > 0 ? ceil_div(a->length, conv_tile(a)) : 1; }
// backward: each block's partial sums are K + 1 values a channel; two blocks to a compute unit, over the channels' groups
static int64_t conv_blocks(const mws_conv_args *a) {
    int64_t need = ceil_div(a->batch * conv_tiles(a), 4), groups = ceil_div(a->width, kWave * conv_back_v(a));
    int64_t most = groups < 16 ? 1024 / groups : 64;
    return need < most ? need : most;
}

static int32_t conv_check(const mws_conv_args *a, const char *what, bool backward, bool step) {
    if (a == nullptr) return fail("%s: no arguments", what);
    if (a->type < MWS_F32 || a->type > MWS_F16) return fail("%s: type %d is none of MWS_F32, MWS_BF16, MWS_F16", what, a->type);
    if (a->param_type != MWS_F32 && a->param_type != a->type) return fail("%s: parameters are float or of the activations' type", what);
    if (a->taps < MWS_CONV_MIN_TAPS || a->taps > MWS_CONV_MAX_TAPS) return fail("%s: %d taps are not within %d .. %d", what, a->taps, MWS_CONV_MIN_TAPS, MWS_CONV_MAX_TAPS);
    if (a->width < 1 || a->width > (1 << 22)) return fail("%s: width %d", what, a->width);
    if (a->batch < 0 || a->length < 0 || a->batch > (1 << 30) || a->length > (1 << 30) || a->batch * (a->length + 1) > ((int64_t)1 << 33)) return fail("%s: %lld rows of %lld tokens", what, (long long)a->batch, (long long)a->length);
    if (a->weight == nullptr) return fail("%s: weight is NULL", what);
    if (step && a->length != 1) return fail("%s: one token at a time", what);
    if (a->batch == 0) return 0;
    if (a->length > 0 && a->x == nullptr) return fail("%s: x is NULL", what);
    if (!backward && a->length > 0 && a->y == nullptr) return fail("%s: y is NULL", what);
    if (backward && a->length > 0 && a->dy == nullptr) return fail("%s: dy is NULL", what);
    if (step && (a->state == nullptr || a->last == nullptr)) return fail("%s: the state is NULL", what);
    return 0;
}

// whether the launches can count their threads
static int32_t conv_fits(const mws_conv_args *a, const char *what, bool backward, bool step) {
    const int v = step && a->width % conv_v(a) != 0 ? 1 : conv_v(a);
    bool all = step       ? fits(ceil_div(step_lanes(a->batch, ceil_div(a->width, v), kStepRows) * ceil_div(a->width, v), 256), 256)
               : backward ? fits(ceil_div((int64_t)(a->taps + 1) * a->width, 32), 1024)
                          : fits(ceil_div(a->batch * conv_tiles(a), 4), 256);
    return all ? 0 : fail("%s: %lld rows of %lld tokens and %d channels are more than one launch can count", what, (long long)a->batch, (long long)a->length, a->width);
}

static ConvArgs conv_device(const mws_conv_args *a) {
    ConvArgs d = {};
    d.x = a->x, d.weight = a->weight, d.bias = a->bias, d.state = a->state, d.dy = a->dy, d.dlast = a->dlast;
    d.reset = a->reset, d.lengths = a->lengths, d.y = a->y, d.last = a->last, d.dx = a->dx, d.dstate = a->dstate;
    d.batch = a->batch, d.length = a->length, d.tile = conv_tile(a);
    d.tiles = conv_tiles(a);
    d.x_batch = a->x_batch, d.x_time = a->x_time, d.dy_batch = a->dy_batch, d.dy_time = a->dy_time;
    d.reset_batch = a->reset_batch, d.reset_time = a->reset_time;
    d.width = a->width, d.wide = a->param_type == MWS_F32;
    return d;
}

enum { kForward, kBackward, kStep };
template <class T, int V, int K> static void conv_go(const mws_conv_args *a, const ConvArgs &d, int what, hipStream_t stream) {
    unsigned groups = (unsigned)ceil_div(a->width, kWave * V);
    if constexpr (V <= 4) {
        if (what == kBackward) {
            hipLaunchKernelGGL((conv_backward<T, V, K>), dim3((unsigned)conv_blocks(a), groups), dim3(256), 0, stream, d);
            return;
        }
    }
    if (what == kForward) hipLaunchKernelGGL((conv_forward<T, V, K>), dim3((unsigned)ceil_div(d.batch * d.tiles, 4), groups), dim3(256), 0, stream, d);
    else {
        int64_t across = ceil_div(a->width, V), each = step_lanes(d.batch, across, kStepRows);
        hipLaunchKernelGGL((conv_step<T, V, K>), dim3((unsigned)ceil_div(each * across, 256)), dim3(256), 0, stream, d, across, each);
    }
}
template <class T, int V> static void conv_taps(const mws_conv_args *a, const ConvArgs &d, int what, hipStream_t stream) {
    if (a->taps == 2) conv_go<T, V, 2>(a, d, what, stream);
    else if (a->taps == 3) conv_go<T, V, 3>(a, d, what, stream);
    else conv_go<T, V, 4>(a, d, what, stream);
}
template <class T, int V> static void conv_width(const mws_conv_args *a, const ConvArgs &d, int what, hipStream_t stream) {
    if (what == kBackward) {
        if (a->width >= 4) conv_taps<T, 4>(a, d, what, stream);
        else conv_taps<T, 1>(a, d, what, stream);
    } else if (what == kStep ? a->width % V == 0 : a->width >= V) conv_taps<T, V>(a, d, what, stream);
    else conv_taps<T, 1>(a, d, what, stream);
}
static void conv_run(const mws_conv_args *a, const ConvArgs &d, int what, hipStream_t stream) {
    if (a->type == MWS_F32) conv_width<F32, 4>(a, d, what, stream);
    else if (a->type == MWS_BF16) conv_width<BF16, 8>(a, d, what, stream);
    else conv_width<F16, 8>(a, d, what, stream);
}
}  // namespace mws

using namespace mws;

extern "C" int32_t mws_conv_forward(const mws_conv_args *a, void *stream) {
    if (int32_t e = conv_check(a, "mws_conv_forward", false, false)) return e;
    if (a->batch == 0) return 0;
    if (int32_t e = conv_fits(a, "mws_conv_forward", false, false)) return e;
    conv_run(a, conv_device(a), kForward, (hipStream_t)stream);
    return launched("mws_conv_forward");
}

extern "C" int64_t mws_conv_workspace(const mws_conv_args *a) {
    if (int32_t e = conv_check(a, "mws_conv_workspace", true, false)) return e;
    return a->dweight != nullptr || a->dbias != nullptr ? conv_blocks(a) * (a->taps + 1) * a->width * (int64_t)sizeof(float) : 0;
}

extern "C" int32_t mws_conv_backward(const mws_conv_args *a, void *stream) {
    if (int32_t e = conv_check(a, "mws_conv_backward", true, false)) return e;
    int64_t need = mws_conv_workspace(a);
    if (a->workspace_bytes < need || (need > 0 && a->workspace == nullptr)) return fail("mws_conv_backward: the workspace needs %lld bytes", (long long)need);
    if (int32_t e = conv_fits(a, "mws_conv_backward", true, false)) return e;
    ConvArgs d = conv_device(a);
    bool params = a->dweight != nullptr || a->dbias != nullptr;
    d.part = params ? (float *)a->workspace : nullptr;
    int64_t blocks = conv_blocks(a);
    if (blocks > 0) conv_run(a, d, kBackward, (hipStream_t)stream);
    if (params) {
        ConvOut out = {a->dweight, a->dbias, a->width, a->taps, a->type, a->param_type == MWS_F32};
        launch_sum_parts((const float *)a->workspace, (int)blocks, (int64_t)(a->taps + 1) * a->width, out, (hipStream_t)stream);
    }
    return launched("mws_conv_backward");
}

extern "C" int32_t mws_conv_step(const mws_conv_args *a, void *stream) {
    if (int32_t e = conv_check(a, "mws_conv_step", false, true)) return e;
    if (a->batch == 0) return 0;
    if (int32_t e = conv_fits(a, "mws_conv_step", false, true)) return e;
    conv_run(a, conv_device(a), kStep, (hipStream_t)stream);
    return launched("mws_conv_step");
}
