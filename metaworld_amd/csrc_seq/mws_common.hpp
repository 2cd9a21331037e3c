// mws_common.hpp -- types, vector loads, wave reductions and the sum over partial results that the sequence operators share.
#pragma once
#include <hip/hip_runtime.h>
#include <cstdint>
#include <cstdio>
#include "../../include/mwseq.h"

namespace mws {

constexpr int kWave = 64;
constexpr int kSimds = 1024;          // 256 compute units with four SIMDs each

// ---- element types: arithmetic is float, a value is rounded to the nearest once, where it is stored ----
struct F32 { using raw = float; };
struct BF16 { using raw = uint16_t; };
struct F16 { using raw = uint16_t; };

template <class T> __device__ __forceinline__ float up(typename T::raw v);
template <> __device__ __forceinline__ float up<F32>(float v) { return v; }
template <> __device__ __forceinline__ float up<BF16>(uint16_t v) { return __builtin_bit_cast(float, (uint32_t)v << 16); }
template <> __device__ __forceinline__ float up<F16>(uint16_t v) { return (float)__builtin_bit_cast(_Float16, v); }
template <class T> __device__ __forceinline__ typename T::raw down(float v);
template <> __device__ __forceinline__ float down<F32>(float v) { return v; }
template <> __device__ __forceinline__ uint16_t down<BF16>(float v) { return __builtin_bit_cast(uint16_t, (__bf16)v); }
template <> __device__ __forceinline__ uint16_t down<F16>(float v) { return __builtin_bit_cast(uint16_t, (_Float16)v); }

// V values at any address: the memory pipeline takes unaligned vector accesses to global memory, so that odd widths and strides
// keep 16-byte loads
template <class T, int V> struct Vec {
    typename T::raw v[V];
};
template <class T, int V> __device__ __forceinline__ Vec<T, V> load(const typename T::raw *p) {
    Vec<T, V> r;
    __builtin_memcpy(&r, p, sizeof(r));
    return r;
}
template <class T, int V> __device__ __forceinline__ void store(typename T::raw *p, const Vec<T, V> &r) { __builtin_memcpy(p, &r, sizeof(r)); }
// n of them (0 <= n <= V), the others zero
template <class T, int V> __device__ __forceinline__ Vec<T, V> load_some(const typename T::raw *p, int n) {
    if (n >= V) return load<T, V>(p);
    Vec<T, V> r;
#pragma unroll
    for (int i = 0; i < V; i++) r.v[i] = i < n ? p[i] : (typename T::raw)0;
    return r;
}
template <class T, int V> __device__ __forceinline__ void store_some(typename T::raw *p, const Vec<T, V> &r, int n) {
    if (n >= V) {
        store<T, V>(p, r);
        return;
    }
#pragma unroll
    for (int i = 0; i < V; i++)
        if (i < n) p[i] = r.v[i];
}

// ---- functions: hardware exp2 / log2 / reciprocal (each within one unit in the last place) ----
constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;
__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float exp_(float x) { return exp2_(x * kLog2e); }
__device__ __forceinline__ float rcp_(float x) { return __builtin_amdgcn_rcpf(x); }
__device__ __forceinline__ float sigmoid_(float x) { return rcp_(1.0f + exp_(-x)); }

// ---- lanes of a wave ----
__device__ __forceinline__ void swap32(float &x, float &y) {         // the upper half of x and the lower half of y
    auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, x), __builtin_bit_cast(unsigned, y), false, false);
    unsigned r0 = r[0], r1 = r[1];       // (a bit cast of an element itself takes the vector's first)
    x = __builtin_bit_cast(float, r0), y = __builtin_bit_cast(float, r1);
}
__device__ __forceinline__ void swap16(float &x, float &y) {         // the odd rows (of 16 lanes) of x and the even rows of y
    auto r = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(unsigned, x), __builtin_bit_cast(unsigned, y), false, false);
    unsigned r0 = r[0], r1 = r[1];
    x = __builtin_bit_cast(float, r0), y = __builtin_bit_cast(float, r1);
}
template <int CTRL> __device__ __forceinline__ float dpp(float x) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), CTRL, 0xf, 0xf, true));
}
constexpr int kRor8 = 0x128, kHalfMirror = 0x141, kQuad2 = 0x4E, kQuad1 = 0xB1;    // the lane 8 on in its row; 7 - lane in its half row; lane ^ 2; lane ^ 1

// the sum over groups of N neighbouring lanes, to all of them, in vector instructions alone (a sum of 64 through shared memory's
// permutation takes six round trips of it: layer norm of 262144 x 512 bf16 144 us with that, 133 us with this)
template <int N> __device__ __forceinline__ float lane_sum(float v) {
    static_assert(N >= 1 && N <= 64 && (N & (N - 1)) == 0, "a power of two");
    if constexpr (N >= 2) v += dpp<kQuad1>(v);
    if constexpr (N >= 4) v += dpp<kQuad2>(v);
    if constexpr (N >= 8) v += dpp<kHalfMirror>(v);
    if constexpr (N >= 16) v += dpp<kRor8>(v);
    if constexpr (N >= 32) {
        float w = v;
        swap16(v, w);
        v += w;
    }
    if constexpr (N >= 64) {
        float w = v;
        swap32(v, w);
        v += w;
    }
    return v;
}

__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

// ---- the sum over partial results: part[count][columns] -> out(column, sum), always in the same order ----
// One block sums 32 columns: 32 groups of threads take every 32nd row, the groups' sums meet in shared memory.  Bound by latency,
// not by bytes: 32 x 32 threads keep count / 32 dependent loads per thread.
template <class Out> __global__ __launch_bounds__(1024) void sum_parts(const float *__restrict__ part, int count, int64_t columns, Out out) {
    __shared__ float meet[32][33];
    int c = threadIdx.x & 31, r = threadIdx.x >> 5;
    int64_t col = (int64_t)blockIdx.x * 32 + c;
    float s0 = 0, s1 = 0, s2 = 0, s3 = 0;
    if (col < columns) {
        int k = r;
        for (; k + 96 < count; k += 128) {
            s0 += part[(int64_t)k * columns + col];
            s1 += part[(int64_t)(k + 32) * columns + col];
            s2 += part[(int64_t)(k + 64) * columns + col];
            s3 += part[(int64_t)(k + 96) * columns + col];
        }
        for (; k < count; k += 32) s0 += part[(int64_t)k * columns + col];
    }
    meet[r][c] = (s0 + s1) + (s2 + s3);
    __syncthreads();
    // 32 sums of 32: each wave takes two columns of the transposed square
    float v = meet[c][r];
    v = lane_sum<32>(v);
    int64_t mine = (int64_t)blockIdx.x * 32 + r;
    if (c == 0 && mine < columns) out(mine, v);
}

template <class Out> inline void launch_sum_parts(const float *part, int count, int64_t columns, Out out, hipStream_t stream) {
    if (columns > 0) hipLaunchKernelGGL((sum_parts<Out>), dim3((unsigned)((columns + 31) / 32)), dim3(1024), 0, stream, part, count, columns, out);
}

// ---- host: how many rows of one token a lane takes, so that its parameters are read once: up to `most`, as long as a quarter of the card's
// places for waves stay filled.  Returns the number of lanes over the rows ----
inline int64_t step_lanes(int64_t rows, int64_t lanes_of_row, int most) {
    int64_t fill = (int64_t)kSimds * 2 * kWave, few = (rows + most - 1) / most, wanted = (fill + lanes_of_row - 1) / lanes_of_row;
    int64_t lanes = wanted > few ? wanted : few;
    return lanes < rows ? lanes : rows;
}

// ---- host: errors ----
extern thread_local char g_error[256];
template <class... A> inline int32_t fail(const char *form, A... a) {
    snprintf(g_error, sizeof(g_error), form, a...);
    return MWS_ARGUMENT;
}
inline int32_t fail(const char *text) { return fail("%s", text); }
inline int32_t launched(const char *what) {
    hipError_t e = hipGetLastError();
    if (e == hipSuccess) return 0;
    snprintf(g_error, sizeof(g_error), "%s: %s", what, hipGetErrorString(e));
    return MWS_LAUNCH;
}
inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
// a launch counts its threads along an axis in 32 bits, its blocks in 31
inline bool fits(int64_t blocks, int threads) { return blocks <= 0x7fffffff && blocks * threads <= 0xffffffffLL; }

}  // namespace mws
