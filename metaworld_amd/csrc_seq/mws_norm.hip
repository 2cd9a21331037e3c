// mws_norm.hip -- layer norm, forward and backward.
//
//   m = mean x, v = mean (x - m)^2, r = (v + eps)^-1/2, n = (x - m) r, y = n w + b
//   g = dy w, dx = r (g - mean g - n mean(g n)), dw = sum over rows of dy n, db = sum over rows of dy
//
// Bound by memory, 262144 x 512 bf16 forward in 121 us (4.4 TB/s; a copy of 4 GiB reaches 4.8), backward in 170 us (4.7 TB/s): one
// pass over the data.  A row stays in the registers of TPR threads (V values to a 16-byte load, PER loads to
// a thread), the variance is taken from the centred values (two sums over the lanes, no difference of large squares), and the
// parameters stay in registers while a block walks over its rows.  The backward pass takes mean and r anew from the row it reads
// anyway, so the forward pass stores nothing for it; each thread sums its columns' dw and db over the block's rows, blocks leave
// partial sums, and sum_parts adds them in a fixed order.
#include "mws_common.hpp"

namespace mws {
thread_local char g_error[256] = "";

struct NormArgs {
    const void *x, *weight, *bias, *dy;
    void *y, *dx;
    float *part;                 // [blocks][2][width]
    int64_t rows, x_stride, dy_stride;
    int width;
    bool wide;                   // float parameters
    float share, eps;            // 1 / width
};

// the sum over a row's threads, to all of them.  Over several waves through shared memory: `turn` alternates between its halves, so
// that one barrier is enough (who writes a half again has passed the barrier after its last reading)
template <int TPR> __device__ __forceinline__ float row_sum(float v, float (*meet)[16], int &turn) {
    v = lane_sum<(TPR < kWave ? TPR : kWave)>(v);
    if constexpr (TPR > kWave) {
        if (threadIdx.x % kWave == 0) meet[turn][threadIdx.x / kWave] = v;
        __syncthreads();
        v = 0;
#pragma unroll
        for (int k = 0; k < TPR / kWave; k++) v += meet[turn][k];
        turn ^= 1;
    }
    return v;
}
template <int TPR> __device__ __forceinline__ void row_sums(float &v, float &u, float (*meet)[16], float (*meet2)[16], int &turn) {
    v = lane_sum<(TPR < kWave ? TPR : kWave)>(v), u = lane_sum<(TPR < kWave ? TPR : kWave)>(u);
    if constexpr (TPR > kWave) {
        if (threadIdx.x % kWave == 0) meet[turn][threadIdx.x / kWave] = v, meet2[turn][threadIdx.x / kWave] = u;
        __syncthreads();
        v = u = 0;
#pragma unroll
        for (int k = 0; k < TPR / kWave; k++) v += meet[turn][k], u += meet2[turn][k];
        turn ^= 1;
    }
}

template <class T, int V, int PER, int TPR> struct Row {
    float v[PER * V];
    __device__ __forceinline__ void read(const typename T::raw *p, int lane, int width) {
#pragma unroll
        for (int k = 0; k < PER; k++) {
            int col = (k * TPR + lane) * V;
            Vec<T, V> r = load_some<T, V>(p + (col < width ? col : 0), width - col);
#pragma unroll
            for (int i = 0; i < V; i++) v[k * V + i] = up<T>(r.v[i]);
        }
    }
    __device__ __forceinline__ void write(typename T::raw *p, int lane, int width) const {
#pragma unroll
        for (int k = 0; k < PER; k++) {
            int col = (k * TPR + lane) * V;
            Vec<T, V> r;
#pragma unroll
            for (int i = 0; i < V; i++) r.v[i] = down<T>(v[k * V + i]);
            if (col < width) store_some<T, V>(p + col, r, width - col);
        }
    }
    // whole vectors: a condition for each value is a branch with a wait of its own, and every block begins with them (8000 x 512 bf16
    // forward 6 us, 11 us value by value)
    __device__ __forceinline__ void read_param(const void *p, int lane, int width, bool wide, float otherwise) {
#pragma unroll
        for (int k = 0; k < PER; k++) {
            int col = (k * TPR + lane) * V, from = col < width ? col : 0, n = width - col;
            if (p == nullptr) {
#pragma unroll
                for (int i = 0; i < V; i++) v[k * V + i] = otherwise;
            } else if (wide) {
                Vec<F32, V> r = load_some<F32, V>((const float *)p + from, n);
#pragma unroll
                for (int i = 0; i < V; i++) v[k * V + i] = r.v[i];
            } else {
                Vec<T, V> r = load_some<T, V>((const typename T::raw *)p + from, n);
#pragma unroll
                for (int i = 0; i < V; i++) v[k * V + i] = up<T>(r.v[i]);
            }
        }
    }
    // centres the row and returns r; columns past the width stay zero
    __device__ __forceinline__ float centre(int lane, int width, float share, float eps, float (*meet)[16], int &turn) {
        float s = 0;
#pragma unroll
        for (int k = 0; k < PER * V; k++) s += v[k];
        s = row_sum<TPR>(s, meet, turn);
        // the quotient to the last bit (a product and the correction of its error): a row of equal values has to come out as zeros,
        // and 1 / sqrt(eps) times an error of the mean is seen
        float mean = s * share, q = 0;
        mean = __builtin_fmaf(__builtin_fmaf(-mean, (float)width, s), share, mean);
#pragma unroll
        for (int k = 0; k < PER; k++)
#pragma unroll
            for (int i = 0; i < V; i++) {
                int col = (k * TPR + lane) * V + i;
                float c = col < width ? v[k * V + i] - mean : 0.0f;
                v[k * V + i] = c;
                q += c * c;
            }
        float v = row_sum<TPR>(q, meet, turn) * share + eps;
        // (the hardware's 1 / sqrt takes numbers below the smallest normal one as zeros: they are scaled)
        return v < 0x1p-96f ? __builtin_amdgcn_rsqf(v * 0x1p64f) * 0x1p32f : __builtin_amdgcn_rsqf(v);
    }
};

template <class T, int V, int PER, int TPR> __global__ __launch_bounds__(TPR > kWave ? TPR : 256) void norm_forward(NormArgs a) {
    constexpr int kRows = TPR <= kWave ? 256 / TPR : 1;      // rows of one block at a time
    __shared__ float meet[2][16];
    int lane = threadIdx.x % TPR, sub = threadIdx.x / TPR, turn = 0;
    Row<T, V, PER, TPR> w, b, x;
    w.read_param(a.weight, lane, a.width, a.wide, 1.0f);
    b.read_param(a.bias, lane, a.width, a.wide, 0.0f);
    for (int64_t row0 = (int64_t)blockIdx.x * kRows; row0 < a.rows; row0 += (int64_t)gridDim.x * kRows) {
        int64_t row = row0 + sub;
        bool on = row < a.rows;
        x.read((const typename T::raw *)a.x + (on ? row : a.rows - 1) * a.x_stride, lane, a.width);
        float r = x.centre(lane, a.width, a.share, a.eps, meet, turn);
#pragma unroll
        for (int k = 0; k < PER * V; k++) x.v[k] = x.v[k] * r * w.v[k] + b.v[k];
        if (on) x.write((typename T::raw *)a.y + row * a.width, lane, a.width);
    }
}

template <class T, int V, int PER, int TPR> __global__ __launch_bounds__(TPR > kWave ? TPR : 256) void norm_backward(NormArgs a) {
    constexpr int kRows = TPR <= kWave ? 256 / TPR : 1;
    __shared__ float meet[2][16], meet2[2][16];
    int lane = threadIdx.x % TPR, sub = threadIdx.x / TPR, turn = 0;
    Row<T, V, PER, TPR> w, x, g;
    float dw[PER * V], db[PER * V];
#pragma unroll
    for (int k = 0; k < PER * V; k++) dw[k] = db[k] = 0;
    w.read_param(a.weight, lane, a.width, a.wide, 1.0f);
    for (int64_t row0 = (int64_t)blockIdx.x * kRows; row0 < a.rows; row0 += (int64_t)gridDim.x * kRows) {
        int64_t row = row0 + sub;
        bool on = row < a.rows;
        int64_t at = on ? row : a.rows - 1;
        x.read((const typename T::raw *)a.x + at * a.x_stride, lane, a.width);
        g.read((const typename T::raw *)a.dy + at * a.dy_stride, lane, a.width);
        float r = x.centre(lane, a.width, a.share, a.eps, meet, turn), s = 0, q = 0;
#pragma unroll
        for (int k = 0; k < PER * V; k++) {
            float n = x.v[k] * r, d = g.v[k];
            x.v[k] = n;
            dw[k] += on ? d * n : 0.0f;
            db[k] += on ? d : 0.0f;
            d *= w.v[k];
            g.v[k] = d;
            s += d;                    // columns past the width were read as zeros
            q += d * n;
        }
        row_sums<TPR>(s, q, meet, meet2, turn);
        s *= a.share;
        q *= a.share;
        if (a.dx != nullptr) {
#pragma unroll
            for (int k = 0; k < PER * V; k++) x.v[k] = r * (g.v[k] - s - x.v[k] * q);
            if (on) x.write((typename T::raw *)a.dx + row * a.width, lane, a.width);
        }
    }
    if (a.part == nullptr) return;
    float *part = a.part + (int64_t)blockIdx.x * 2 * a.width;
    if constexpr (kRows > 1) {
        // the block's sums: the rows that it took side by side meet in shared memory, behind one barrier for all columns
        __shared__ float pool[2 * PER * V][256];
#pragma unroll
        for (int k = 0; k < PER * V; k++) pool[k][threadIdx.x] = dw[k], pool[PER * V + k][threadIdx.x] = db[k];
        __syncthreads();
        for (int r = sub; r < 2 * PER * V; r += kRows) {
            float v = 0;
#pragma unroll
            for (int j = 0; j < kRows; j++) v += pool[r][j * TPR + lane];
            int k = r % (PER * V), col = ((k / V) * TPR + lane) * V + k % V;
            if (col < a.width) part[r / (PER * V) * a.width + col] = v;
        }
    } else
#pragma unroll
        for (int k = 0; k < PER * V; k++) {
            int col = ((k / V) * TPR + lane) * V + k % V;
            if (col < a.width) part[col] = dw[k], part[a.width + col] = db[k];
        }
}

struct NormOut {
    void *dweight, *dbias;
    int width, type;
    bool wide;
    __device__ void operator()(int64_t col, float v) const {
        void *to = col < width ? dweight : dbias;
        int64_t at = col < width ? col : col - width;
        if (to == nullptr) return;
        if (wide || type == MWS_F32) ((float *)to)[at] = v;
        else if (type == MWS_BF16) ((uint16_t *)to)[at] = down<BF16>(v);
        else ((uint16_t *)to)[at] = down<F16>(v);
    }
};

// Threads of a row: eight values each from 1025 columns on (16384 x 4096 bf16 forward 53 us, backward 115 us; with sixteen 71 and
// 160 us when with eight it was 65 and 116).  Blocks walk over the rows, 4096 waves in all (262144 x 512 bf16 forward 123 us, backward 170 us; with twice as many 128
// and 195 us); twice that forward in blocks of 1024 threads, two of which fit a compute unit (4000 x 16384 fp32 113 us, not 182).  Beyond 8192 columns a thread has sixteen again, and backward some registers
// do not fit (bf16 28, fp16 16 spilled; 4000 x 16384 bf16 backward 140 us, 2.8 TB/s; fp32 183 us, 4.3 TB/s).
static int norm_rows(int tpr) { return tpr <= kWave ? 256 / tpr : 1; }
static int norm_tpr(const mws_norm_args *a) {
    int v = a->type == MWS_F32 ? 4 : 8, w = a->width;
    return w <= 8 * v ? 8 : w <= 16 * v ? 16 : w <= 32 * v ? 32 : w <= 1024 ? 64 : w <= 2048 ? 256 : w <= 4096 ? 512 : 1024;
}
static int64_t norm_blocks(const mws_norm_args *a, bool backward) {
    int tpr = norm_tpr(a);
    int64_t most = tpr <= 256 ? 1024 : tpr == 512 || !backward ? 512 : 256, need = ceil_div(a->rows, norm_rows(tpr));
    return need < most ? need : most;
}

template <class T, int V> static void norm_launch(const mws_norm_args *a, const NormArgs &d, bool backward, hipStream_t stream) {
    dim3 grid((unsigned)norm_blocks(a, backward));
    int w = a->width;
#define MWS_GO(PER, TPR)                                                                                                            \
    do {                                                                                                                            \
        if (backward) hipLaunchKernelGGL((norm_backward<T, V, PER, TPR>), grid, dim3(TPR > kWave ? TPR : 256), 0, stream, d);       \
        else hipLaunchKernelGGL((norm_forward<T, V, PER, TPR>), grid, dim3(TPR > kWave ? TPR : 256), 0, stream, d);                 \
    } while (0)
    constexpr int P = 16 / V;                // sixteen values of a row to a thread at most, eight in blocks of several waves: five rows' worth of registers backward
    switch (norm_tpr(a)) {
        case 8: MWS_GO(1, 8); break;
        case 16: MWS_GO(1, 16); break;
        case 32: MWS_GO(1, 32); break;
        case 64:
            if (w <= 64 * V) MWS_GO(1, 64);
            else if (w <= 128 * V) MWS_GO(2, 64);
            else MWS_GO(P, 64);
            break;
        case 256: MWS_GO(P / 2, 256); break;
        case 512: MWS_GO(P / 2, 512); break;
        default:
            if (w <= 8192) MWS_GO(P / 2, 1024);
            else MWS_GO(P, 1024);
    }
#undef MWS_GO
}

static int32_t norm_check(const mws_norm_args *a, bool backward) {
    if (a == nullptr) return fail("mws_norm: no arguments");
    if (a->type < MWS_F32 || a->type > MWS_F16) return fail("mws_norm: type %d is none of MWS_F32, MWS_BF16, MWS_F16", a->type);
    if (a->param_type != MWS_F32 && a->param_type != a->type) return fail("mws_norm: parameters are float or of the activations' type");
    if (a->rows < 0 || a->rows > ((int64_t)1 << 40)) return fail("mws_norm: %lld rows", (long long)a->rows);
    if (a->width < 1 || a->width > MWS_NORM_MAX_WIDTH) return fail("mws_norm: width %d is not within 1 .. %d", a->width, MWS_NORM_MAX_WIDTH);
    if (!(a->eps >= 0)) return fail("mws_norm: eps is negative or no number");
    if (a->rows > 0 && a->x == nullptr) return fail("mws_norm: x is NULL");
    if (!backward && a->rows > 0 && a->y == nullptr) return fail("mws_norm: y is NULL");
    if (backward && a->rows > 0 && a->dy == nullptr) return fail("mws_norm: dy is NULL");
    return 0;
}

static NormArgs norm_device(const mws_norm_args *a) {
    NormArgs d = {a->x, a->weight, a->bias, a->dy, a->y, a->dx, nullptr, a->rows, a->x_stride, a->dy_stride, a->width, a->param_type == MWS_F32, 1.0f / (float)a->width, a->eps};
    return d;
}
static void norm_run(const mws_norm_args *a, const NormArgs &d, bool backward, hipStream_t stream) {
    if (a->type == MWS_F32) norm_launch<F32, 4>(a, d, backward, stream);
    else if (a->type == MWS_BF16) norm_launch<BF16, 8>(a, d, backward, stream);
    else norm_launch<F16, 8>(a, d, backward, stream);
}
}  // namespace mws

using namespace mws;

extern "C" const char *mws_last_error(void) { return g_error; }
extern "C" int64_t mws_sizeof(int32_t which) {
    return which == 0 ? (int64_t)sizeof(mws_norm_args) : which == 1 ? (int64_t)sizeof(mws_conv_args) : which == 2 ? (int64_t)sizeof(mws_scan_args) : -1;
}

extern "C" int32_t mws_norm_forward(const mws_norm_args *a, void *stream) {
    if (int32_t e = norm_check(a, false)) return e;
    if (a->rows == 0) return 0;
    norm_run(a, norm_device(a), false, (hipStream_t)stream);
    return launched("mws_norm_forward");
}

extern "C" int64_t mws_norm_workspace(const mws_norm_args *a) {
    if (int32_t e = norm_check(a, true)) return e;
    return a->dweight != nullptr || a->dbias != nullptr ? norm_blocks(a, true) * 2 * a->width * (int64_t)sizeof(float) : 0;
}

extern "C" int32_t mws_norm_backward(const mws_norm_args *a, void *stream) {
    if (int32_t e = norm_check(a, true)) return e;
    int64_t need = mws_norm_workspace(a);
    if (a->workspace_bytes < need || (need > 0 && a->workspace == nullptr)) return fail("mws_norm_backward: the workspace needs %lld bytes", (long long)need);
    NormArgs d = norm_device(a);
    bool params = a->dweight != nullptr || a->dbias != nullptr;
    d.part = params ? (float *)a->workspace : nullptr;
    if (a->rows > 0 && (params || a->dx != nullptr)) norm_run(a, d, true, (hipStream_t)stream);
    if (params) {
        NormOut out = {a->dweight, a->dbias, a->width, a->type, a->param_type == MWS_F32};
        launch_sum_parts((const float *)a->workspace, (int)norm_blocks(a, true), 2 * (int64_t)a->width, out, (hipStream_t)stream);
    }
    return launched("mws_norm_backward");
}
