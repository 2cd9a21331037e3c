// mws_scan.hip -- the selective state space scan: forward, backward, one token.
//
//   d_t = softplus(dt_t + dt_bias), a_t = exp(d_t A), h_t = a_t h_{t-1} + d_t u_t B_t, o_t = C_t . h_t + D u_t, y_t = o_t silu(z_t)
//   do = dy silu(z), g_t = do_t C_t + a_{t+1} g_{t+1}
//   dC_t = sum over channels of do h_t, dB_t = sum over channels of g d u, du = D do + d (g . B), dz = dy o silu'(z)
//   dd_t = u (g . B) + g . (A a_t h_{t-1}), ddt = dd sigmoid(dt + dt_bias), dA = sum over tokens of g d a_t h_{t-1}
//
// where an episode begins, a_t counts as zero.
//
// A lane is a channel with all its states in registers, so that a token's B and C are the same for the whole wave: they come in
// scalar registers, from a small copy in float, [token][B | C][states], that `spread` makes first (128 bytes a token next to the
// channels' 8 bytes each).  A wave walks along the time axis; u, dt, z and y are read and written in order of channels.
// Bound by the vector unit: per value and state one exp (two issue slots) and four multiplications or additions forward, 147
// slots a token and wave with 16 states.  2048 x 64 x 512 x 16 bf16 forward in 267 us with the copy of B and C (7 us), 251 us of them slots; the
// memory would allow 140.
//
// Where batch x channels leave the card empty, the time axis is cut into segments: scan_segment takes each
// segment's end state from zero and its sum of d (the product of its a is exp(A sum d)), scan_join runs over the segments, and the
// scan itself starts every segment from its joined state.  The same holds for g, from the end.
#include "mws_common.hpp"

namespace mws {

// Tokens are walked in groups of kGroup, whose episodes' beginnings are one mask.  Every kKept-th token's state is kept for the
// backward pass, which holds what lies between two of them in registers (states x tokens = 128); segments begin at these tokens.
// lanes_of: a block's channels at most.
constexpr int kGroup = 32, kKept = 8;
constexpr int lanes_of(int ns) { return ns >= 32 ? 128 : 256; }

struct ScanArgs {
    const void *u, *dt, *z, *dy;
    const float *A, *D, *dt_bias, *state, *dlast;
    const uint8_t *reset;
    const int32_t *lengths;
    void *y, *du, *ddt, *dz;
    float *last, *kept, *dstate;
    const float *bc;             // [batch][length][2][NS]
    float *seg, *sum;            // [batch][segments][NS][width] states, [batch][segments][width] sums of d (negative: cut by an episode's beginning)
    float *part_bc;              // [blocks over channels][batch][length][2 NS]
    float *part;                 // [groups][NS + 2][width]: dA, dD, ddt_bias
    int64_t batch, length, chunks;
    int64_t u_batch, u_time, dt_batch, dt_time, z_batch, z_time, dy_batch, dy_time, reset_batch, reset_time;
    int width, states, across, segments, span, groups;            // across: blocks over the channels; span: tokens of a segment
};

// The channels of a token and of the seven after it as a buffer: the tokens' address is scalar, a lane adds its channel's bytes.  A
// lane past the channels adds kOutside instead: with that it reads zeros and writes nothing, without a branch, as does every lane
// of a tensor that is not there.  (Eight tokens and the channels end below kBytes: MWS_SCAN_MAX_STRIDE.)
constexpr uint32_t kBytes = 0x80000000u, kOutside = 0xC0000000u;
template <class R> struct Line {
    __amdgpu_buffer_rsrc_t r;
    uint32_t stride;
    __device__ __forceinline__ Line(const R *p, int64_t from, int64_t step)
        : r(__builtin_amdgcn_make_buffer_rsrc((void *)(p != nullptr ? p + from : p), 0, (int)(p != nullptr ? kBytes : 0), 0x00020000)), stride((uint32_t)step * (uint32_t)sizeof(R)) {}
    __device__ __forceinline__ R get(uint32_t bytes, int token = 0) const {
        if constexpr (sizeof(R) == 2) return (R)__builtin_amdgcn_raw_buffer_load_b16(r, bytes, token * stride, 0);
        else {
            unsigned v = __builtin_amdgcn_raw_buffer_load_b32(r, bytes, token * stride, 0);
            return __builtin_bit_cast(R, v);
        }
    }
    __device__ __forceinline__ void put(R v, uint32_t bytes, int token = 0) const {
        if constexpr (sizeof(R) == 2) __builtin_amdgcn_raw_buffer_store_b16(v, r, bytes, token * stride, 0);
        else __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(unsigned, v), r, bytes, token * stride, 0);
    }
};

// The kernel's arguments as they lie in memory, to be read where they are needed: held in registers from the kernel's start on they
// would not fit the scalar registers beside a token's B and C.
using FixedArgs = const __attribute__((address_space(4))) ScanArgs;
__device__ __forceinline__ FixedArgs *fresh_args() {
    FixedArgs *k = (FixedArgs *)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(k));
    return k;
}

__device__ __forceinline__ int64_t row_length(const int32_t *lengths, int64_t b, int64_t length) {
    if (lengths == nullptr) return length;
    int64_t n = lengths[b];
    return n < 0 ? 0 : n > length ? length : n;
}

// log(1 + e^x): with w = 1 + e rounded, log(w) e / (w - 1) undoes the rounding of w; beyond 20 it is x to 32 bits
__device__ __forceinline__ float softplus_(float x) {
    float e = exp_(x), w = 1.0f + e, d = w - 1.0f;
    float l = __builtin_amdgcn_logf(w) * kLn2;
    float r = d == 0.0f ? e : l * (e * rcp_(d));
    return x > 20.0f ? x : r;
}

// bit i: an episode begins at token t0 + i of the group
template <class Args> __device__ __forceinline__ uint32_t group_mask(const Args &a, int64_t b, int64_t t0, int64_t end) {
    if (a.reset == nullptr) return 0;
    int lane = threadIdx.x % kWave;
    int64_t t = t0 + lane;
    return (uint32_t)__ballot(lane < kGroup && t < end && a.reset[b * a.reset_batch + t * a.reset_time] != 0);
}

// ---- B and C in float, padded with zeros to NS states: a thread takes four of them ----
template <class T, int NS> __global__ __launch_bounds__(256) void spread(const void *B, const void *C, float *bc, int64_t batch, int64_t length, int64_t B_batch, int64_t B_time, int64_t C_batch,
                                                                         int64_t C_time, int states) {
    constexpr int kOf = 2 * NS / 4;                   // threads of a token
    int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, t = i / kOf;
    if (t >= length) return;
    int at = (int)(i % kOf) * 4;
    const bool second = at >= NS;
    const int n = second ? at - NS : at;
    for (int64_t b = blockIdx.y; b < batch; b += gridDim.y) {
        const typename T::raw *from = (const typename T::raw *)(second ? C : B) + (second ? b * C_batch + t * C_time : b * B_batch + t * B_time) + n;
        Vec<F32, 4> v;
        if (states % 4 == 0) {
            Vec<T, 4> r = load<T, 4>(n < states ? from : from - n);
#pragma unroll
            for (int k = 0; k < 4; k++) v.v[k] = n < states ? up<T>(r.v[k]) : 0.0f;
        } else
#pragma unroll
            for (int k = 0; k < 4; k++) v.v[k] = n + k < states ? up<T>(from[k]) : 0.0f;
        store<F32, 4>(bc + ((b * length + t) * 2 * NS + at), v);
    }
}

// one token's B and C: the address is the same for the wave and nothing of this kernel writes there, which the constant address
// space says, so that they are scalar loads
using Fixed = const __attribute__((address_space(4))) float;
__device__ __forceinline__ Fixed *fixed(const float *p) { return (Fixed *)(uintptr_t)p; }
//
// They are asked for one step ahead: a step's values are in `hold`'s registers when the next step's loads go out, which then have that
// step's time to arrive (scalar loads may overtake each other, so that a wait is for all of them).  A step is some of a token's states
// of B and C (half of 16), or a whole token's of one of them, since the scalar registers hold no more.  (2048 x 64 x 512 x 16 bf16 with the
// backward pass 1448 us when it was built, 1564 us with a token's values asked for where they are needed; 3 x 5000 x 777 x 12 fp16 109 us, not 117.)
template <int S> struct Pair {
    float B[S], C[S];
    __device__ __forceinline__ void read(Fixed *p, int all) {
#pragma unroll
        for (int n = 0; n < S; n++) B[n] = p[n], C[n] = p[all + n];
    }
    __device__ __forceinline__ void hold() const { asm volatile("" ::"s"(B[0]), "s"(C[0])); }
};
template <int S> struct One {
    float v[S];
    __device__ __forceinline__ void read(Fixed *p) {
#pragma unroll
        for (int n = 0; n < S; n++) v[n] = p[n];
    }
    __device__ __forceinline__ void hold() const { asm volatile("" ::"s"(v[0])); }
};
__device__ __forceinline__ void here_only() { __builtin_amdgcn_sched_barrier(0); }      // nothing moves past this

// a lane's states: NS of them from `first` on, of a row of `states` (padded with zeros).  All loads go out before the first is waited
// for: a condition for each of them would be a branch with a wait of its own, and every wave begins with them (2048 x 64 x 512 x 16
// bf16 forward 271 us when it was built, 314 us so; 405 x 66 x 874 x 32 211 us, not 278).
template <int NS> __device__ __forceinline__ void get_states(const float *row, int states, int first, float (&h)[NS]) {
    if (states % 4 == 0) {
        Vec<F32, 4> r[NS / 4];
#pragma unroll
        for (int k = 0; k < NS / 4; k++) r[k] = load<F32, 4>(row + (first + k * 4 < states ? first + k * 4 : 0));
#pragma unroll
        for (int n = 0; n < NS; n++) h[n] = first + n < states ? r[n / 4].v[n % 4] : 0.0f;
    } else {
#pragma unroll
        for (int n = 0; n < NS; n++) h[n] = row[first + n < states ? first + n : 0];
#pragma unroll
        for (int n = 0; n < NS; n++) h[n] = first + n < states ? h[n] : 0.0f;
    }
}
template <int NS> __device__ __forceinline__ void rates(const ScanArgs &a, uint32_t e, float (&A2)[NS], int first = 0) {       // A / ln 2, for exp2
    get_states<NS>(a.A + (int64_t)e * a.states, a.states, first, A2);
#pragma unroll
    for (int n = 0; n < NS; n++) A2[n] *= kLog2e;
}
template <int NS> __device__ __forceinline__ void first_state(const float *state, const ScanArgs &a, int64_t b, uint32_t e, float (&h)[NS], int first = 0) {
    if (state != nullptr) get_states<NS>(state + (b * a.width + e) * a.states, a.states, first, h);
    else
#pragma unroll
        for (int n = 0; n < NS; n++) h[n] = 0;
}
template <int NS> __device__ __forceinline__ void last_state(float *to, const ScanArgs &a, int64_t b, uint32_t e, const float (&h)[NS], int first = 0) {
    float *row = to + (b * a.width + e) * a.states + first;
    if (a.states % 4 == 0) {
#pragma unroll
        for (int k = 0; k < NS / 4; k++)
            if (first + k * 4 < a.states) store<F32, 4>(row + k * 4, {h[k * 4], h[k * 4 + 1], h[k * 4 + 2], h[k * 4 + 3]});
    } else
#pragma unroll
        for (int n = 0; n < NS; n++)
            if (first + n < a.states) row[n] = h[n];
}
template <int NS> __device__ __forceinline__ void get_row(const float *p, int64_t row, const ScanArgs &a, uint32_t e, float (&h)[NS], int all = NS, int first = 0) {
#pragma unroll
    for (int n = 0; n < NS; n++) h[n] = (p + (row * all + first + n) * a.width)[e];
}
template <int NS> __device__ __forceinline__ void put_row(float *p, int64_t row, const ScanArgs &a, uint32_t e, const float (&h)[NS]) {
#pragma unroll
    for (int n = 0; n < NS; n++) (p + (row * NS + n) * a.width)[e] = h[n];
}

// An episode begins: the states count as zeros.  As a branch, which is hardly ever taken; selections would be there for every token.
template <int NS> __device__ __forceinline__ void forget(float (&h)[NS]) {
#pragma unroll
    for (int n = 0; n < NS; n++) {
        h[n] = 0;
        asm volatile("" : "+v"(h[n]));
    }
}
template <int NS, class Args> __device__ __forceinline__ void kept_row(const Args &a, int64_t row, uint32_t bytes, float (&h)[NS], int all, int first) {
#pragma unroll
    for (int n = 0; n < NS; n++) h[n] = Line<float>(a.kept, (row * all + first + n) * a.width, 0).get(bytes);
}

// Numbers of states are padded to NS with A = B = C = 0, which adds nothing as long as nothing is infinite: infinity times zero is no
// number.  PAD is for states != NS: there no sum over states takes the padding in, and nothing else sees what its states become.
// Forward they are selected to zero; backward a branch leaves out three of the sums' additions, and whole fours of padding altogether.
// (bf16 with it, and summed up with the rest: 1024 x 64 x 512 x 10 forward 120, 123, backward 455, 507 us; 405 x 66 x 874 x 31 forward
// 223, 219, backward 877, 831 us.  With selections backward too 539 and 944 us.)
template <int NS> constexpr int fewest_states() { return NS <= 4 ? 1 : NS <= 8 ? 5 : NS <= 16 ? 9 : 17; }

struct Place {          // what a block of the grid works on
    int64_t b, t0, t1, end;
    uint32_t e;
    int at, seg;
    bool on;
    __device__ __forceinline__ uint32_t bytes(int size) const { return on ? (uint32_t)at * (uint32_t)size : kOutside; }
    template <class Args> __device__ __forceinline__ Place(const Args &a, int64_t item, int part, int lanes = blockDim.x, int mine = threadIdx.x) {
        at = part * lanes + mine;
        on = at < a.width;
        e = on ? at : a.width - 1;
        b = item / a.segments, seg = (int)(item % a.segments);
        end = row_length(a.lengths, b, a.length);
        t0 = (int64_t)seg * a.span, t1 = t0 + a.span < a.length ? t0 + a.span : a.length;
    }
};

constexpr int forward_waves(int ns) { return ns <= 8 ? 8 : ns <= 12 ? 7 : ns <= 16 ? 6 : ns <= 24 ? 4 : 3; }         // of a SIMD: the compiler takes more registers than it needs
template <class T, int NS, bool PAD> __global__ __launch_bounds__(256, forward_waves(NS)) void scan_forward(ScanArgs a) {
    using raw = typename T::raw;
    constexpr int G = 4;
    Place p(a, blockIdx.x / a.across, blockIdx.x % a.across);
    int64_t stop = p.t1 < p.end ? p.t1 : p.end;
    raw *y = (raw *)a.y + (p.b * a.length + p.t0) * a.width;
    bool whole_end = p.end <= p.t1 && (p.end > p.t0 || p.seg == 0);      // the row ends in this segment
    const uint32_t bytes = p.bytes(sizeof(raw));
    if (p.t0 < stop || whole_end) {
        float h[NS], A2[NS];
        rates<NS>(a, p.e, A2);
        if (p.seg == 0) first_state<NS>(a.state, a, p.b, p.e, h);
        else get_row<NS>(a.seg, p.b * a.segments + p.seg, a, p.e, h);
        float D = a.D != nullptr ? a.D[p.e] : 0.0f, bias = a.dt_bias != nullptr ? a.dt_bias[p.e] : 0.0f;
        const raw *u = (const raw *)a.u + p.b * a.u_batch + p.t0 * a.u_time, *dt = (const raw *)a.dt + p.b * a.dt_batch + p.t0 * a.dt_time;
        const raw *z = a.z != nullptr ? (const raw *)a.z + p.b * a.z_batch + p.t0 * a.z_time : nullptr;
        Fixed *bc = fixed(a.bc + (p.b * a.length + p.t0) * 2 * NS);
        float *kept = a.kept != nullptr ? a.kept + (p.b * a.chunks + p.t0 / kKept) * NS * a.width : nullptr;
        constexpr int P = NS > 16 ? 4 : 2, S = NS / P;
        int states = a.states;
        Pair<S> m[2];
        m[0].read(bc, NS);                           // (behind the last token: the next row's, or the workspace's padding)
        auto token = [&](raw ru, raw rd, raw rz, bool first, const Line<raw> &out, int q) __attribute__((always_inline)) {
            float uf = 0, d = 0, du = 0, o = 0, o2 = 0;
#pragma unroll
            for (int k = 0; k < P; k++) {
                m[k & 1].hold();
                if (k + 1 == P) bc += 2 * NS;
                m[~k & 1].read(bc + (k + 1) % P * S, NS);
                here_only();
                if (k == 0) {
                    uf = up<T>(ru), d = softplus_(up<T>(rd) + bias), du = d * uf, o = D * uf;
                    if (first) forget<NS>(h);
                }
                if (PAD) asm volatile("" : "+s"(states));           // no comparison held in registers
#pragma unroll
                for (int i = 0; i < S; i++) {
                    const int n = k * S + i;
                    h[n] = __builtin_fmaf(exp2_(d * A2[n]), h[n], du * m[k & 1].B[i]);
                    if (PAD && n >= fewest_states<NS>()) h[n] = n < states ? h[n] : 0.0f;
                    if (n & 1) o2 = __builtin_fmaf(m[k & 1].C[i], h[n], o2);
                    else o = __builtin_fmaf(m[k & 1].C[i], h[n], o);
                }
                here_only();
            }
            o += o2;
            if (z != nullptr) {
                float zf = up<T>(rz);
                o *= zf * sigmoid_(zf);
            }
            out.put(down<T>(o), bytes, q);
            here_only();
        };
        for (int64_t c0 = p.t0; c0 < stop; c0 += kGroup) {
            uint32_t begins = group_mask(a, p.b, c0, p.end);
            int count = (int)(c0 + kGroup < stop ? kGroup : stop - c0);
            for (int i = 0; i < count; i += G) {
                if (kept != nullptr && i % kKept == 0) {
#pragma unroll
                    for (int n = 0; n < NS; n++) Line<float>(kept, (int64_t)n * a.width, 0).put(h[n], p.bytes(4));
                    kept += (int64_t)NS * a.width;
                }
                Line<raw> lu(u, 0, a.u_time), ld(dt, 0, a.dt_time), lz(z, 0, a.z_time), ly(y, 0, a.width);
                if (i + G <= count) {
                    raw ru[G], rd[G], rz[G];
#pragma unroll
                    for (int q = 0; q < G; q++) ru[q] = lu.get(bytes, q), rd[q] = ld.get(bytes, q), rz[q] = lz.get(bytes, q);
#pragma unroll
                    for (int q = 0; q < G; q++) token(ru[q], rd[q], rz[q], begins >> q & 1, ly, q);
                } else
                    for (int q = 0; i + q < count; q++) token(lu.get(bytes, q), ld.get(bytes, q), lz.get(bytes, q), begins >> q & 1, ly, q);
                begins >>= G;
                u += G * a.u_time, dt += G * a.dt_time, y += G * (int64_t)a.width;
                if (z != nullptr) z += G * a.z_time;
            }
        }
        if (a.last != nullptr && whole_end && p.on) last_state<NS>(a.last, a, p.b, p.e, h);
    }
    y = (raw *)a.y + p.b * a.length * a.width;
    if (p.on)
        for (int64_t t = p.t0 > p.end ? p.t0 : p.end; t < p.t1; t++) (y + t * a.width)[p.e] = down<T>(0.0f);
}

// a segment's end state from zero, and its sum of d
template <class T, int NS> __global__ __launch_bounds__(256) void scan_segment(ScanArgs a) {
    using raw = typename T::raw;
    constexpr int G = 4;
    Place p(a, blockIdx.x / a.across, blockIdx.x % a.across);
    if (p.end <= p.t1) return;           // the row's last segment leaves the row's last state, which scan_forward writes
    const uint32_t bytes = p.bytes(sizeof(raw));
    float h[NS], A2[NS], sum = 0;
    rates<NS>(a, p.e, A2);
#pragma unroll
    for (int n = 0; n < NS; n++) h[n] = 0;
    bool cut = false;
    float bias = a.dt_bias != nullptr ? a.dt_bias[p.e] : 0.0f;
    const raw *u = (const raw *)a.u + p.b * a.u_batch + p.t0 * a.u_time, *dt = (const raw *)a.dt + p.b * a.dt_batch + p.t0 * a.dt_time;
    Fixed *bc = fixed(a.bc + (p.b * a.length + p.t0) * 2 * NS);
    One<NS> B[2];
    B[0].read(bc);
    for (int64_t c0 = p.t0; c0 < p.t1; c0 += kGroup) {        // (a whole segment: the row goes on behind it)
        uint32_t begins = group_mask(a, p.b, c0, p.t1);
        cut = cut || begins != 0;
        const int count = (int)(c0 + kGroup < p.t1 ? kGroup : p.t1 - c0);
        for (int i = 0; i < count; i += G) {
            Line<raw> lu(u, 0, a.u_time), ld(dt, 0, a.dt_time);
            raw ru[G], rd[G];
#pragma unroll
            for (int q = 0; q < G; q++) ru[q] = lu.get(bytes, q), rd[q] = ld.get(bytes, q);
#pragma unroll
            for (int q = 0; q < G; q++) {
                B[q & 1].hold();
                bc += 2 * NS;
                B[~q & 1].read(bc);
                here_only();
                float d = softplus_(up<T>(rd[q]) + bias), x = d * up<T>(ru[q]);
                sum += d;
                if (begins >> q & 1) forget<NS>(h);
#pragma unroll
                for (int n = 0; n < NS; n++) h[n] = __builtin_fmaf(exp2_(d * A2[n]), h[n], x * B[q & 1].v[n]);
                here_only();
            }
            begins >>= G;
            u += G * a.u_time, dt += G * a.dt_time;
        }
    }
    if (p.on) {
        int64_t row = p.b * a.segments + p.seg;
        put_row<NS>(a.seg, row, a, p.e, h);
        a.sum[row * a.width + p.e] = cut ? -1.0f : sum;
    }
}

// what g leaves before a segment's first token, from zero after its last
template <class T, int NS> __global__ __launch_bounds__(256) void scan_segment_back(ScanArgs a) {
    using raw = typename T::raw;
    constexpr int G = 4;
    Place p(a, blockIdx.x / a.across, blockIdx.x % a.across);
    if (p.t0 >= p.end || (p.seg == 0 && a.dstate == nullptr)) return;
    const uint32_t bytes = p.bytes(sizeof(raw));
    int64_t stop = p.t1 < p.end ? p.t1 : p.end;
    float g[NS], A2[NS], sum = 0;
    rates<NS>(a, p.e, A2);
#pragma unroll
    for (int n = 0; n < NS; n++) g[n] = 0;
    bool cut = false;
    const bool gated = a.z != nullptr;
    float bias = a.dt_bias != nullptr ? a.dt_bias[p.e] : 0.0f;
    for (int64_t c0 = p.t0 + (stop - 1 - p.t0) / kGroup * kGroup; c0 >= p.t0; c0 -= kGroup) {
        uint32_t begins = group_mask(a, p.b, c0, stop);
        cut = cut || begins != 0;
        int count = (int)(c0 + kGroup < stop ? kGroup : stop - c0);
        for (int i = (count - 1) / G * G; i >= 0; i -= G) {
            const int64_t t = c0 + i;
            Line<raw> ld((const raw *)a.dt, p.b * a.dt_batch + t * a.dt_time, a.dt_time), ly((const raw *)a.dy, p.b * a.dy_batch + t * a.dy_time, a.dy_time),
                lz((const raw *)a.z, p.b * a.z_batch + t * a.z_time, a.z_time);
            Fixed *bc = fixed(a.bc + (p.b * a.length + t) * 2 * NS);
            raw rd[G], ry[G], rz[G];
            One<NS> C[2];
            C[(G - 1) & 1].read(bc + (G * 2 - 1) * NS);
            const int here = count - i < G ? count - i : G;
#pragma unroll
            for (int q = 0; q < G; q++) {
                int at = q < here ? q : here - 1;
                rd[q] = ld.get(bytes, at), ry[q] = ly.get(bytes, at), rz[q] = lz.get(bytes, at);
            }
#pragma unroll
            for (int q = G - 1; q >= 0; q--) {
                C[q & 1].hold();
                if (q > 0) C[~q & 1].read(bc + (q * 2 - 1) * NS);
                here_only();
                if (q >= here) continue;
                float d = softplus_(up<T>(rd[q]) + bias), o = up<T>(ry[q]);
                if (gated) {
                    float zf = up<T>(rz[q]);
                    o *= zf * sigmoid_(zf);
                }
                sum += d;
#pragma unroll
                for (int n = 0; n < NS; n++) g[n] = exp2_(d * A2[n]) * __builtin_fmaf(o, C[q & 1].v[n], g[n]);
                if (begins >> (i + q) & 1) forget<NS>(g);
                here_only();
            }
        }
    }
    if (p.on) {
        int64_t row = p.b * a.segments + p.seg;
        put_row<NS>(a.seg, row, a, p.e, g);
        a.sum[row * a.width + p.e] = cut ? -1.0f : sum;
    }
}

// Every segment's incoming state, in the place of what it left from zero: forward the state before its first token, backward g after
// its last (from the segment that the row ends in; those behind it are not read).  J threads share a row's chain: each runs over its
// stretch of the segments from zero, then from what the stretches before it make of the row's own state.  (1 x 4096 x 1024 x 16, a
// chain of over a hundred segments: bf16 forward 56 us with eight threads, 71 us with one; where the chains fill the card by themselves one
// is better, 12 x 1000 x 640 x 16 fp32: 88 us, with eight 96 us.)  Chains are counted without the padding of their states, which may differ
// between a pass that is recorded and one that is not: both add in the same order.
static int joiners(int64_t chains, int segments) {
    return segments <= 16 ? 1 : chains * 8 <= 4 * kSimds * kWave ? 8 : chains * 4 <= 4 * kSimds * kWave ? 4 : 1;
}
template <int J> __global__ __launch_bounds__(256) void scan_join(ScanArgs a, int ns, bool backward) {
    constexpr int M = 16, R = 256 / J;               // M segments' values under way at a time: the chain through h does not wait for them
    __shared__ float meet[2][J][R];
    const int c = threadIdx.x % R, mine = threadIdx.x / R;
    int64_t at = (int64_t)blockIdx.x * R + c, all = a.batch * ns * a.width;
    const bool on = at < all;
    if (!on) at = all - 1;
    int e = (int)(at % a.width), n = (int)(at / a.width % ns);
    int64_t b = at / a.width / ns, end = row_length(a.lengths, b, a.length);
    const int last = (int)(end > 0 ? (end - 1) / a.span : 0), per = (last + J) / J, k_from = mine * per, k_to = k_from + per < last + 1 ? k_from + per : last + 1;
    const int asked = backward && a.dstate != nullptr ? last + 1 : last;          // what the last one leaves is dstate
    bool real = n < a.states;
    float A2 = real ? a.A[(int64_t)e * a.states + n] * kLog2e : 0.0f;
    const float *from = backward ? a.dlast : a.state;
    float first = from != nullptr && real ? from[(b * a.width + e) * a.states + n] : 0.0f, left[M], sum[M];
    const int64_t row = b * a.segments;
    auto place = [&](int k) __attribute__((always_inline)) { return row + (backward ? last - k : k); };
    auto read = [&](int k0) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < M; j++) {
            const int k = k0 + j;
            const bool there = k < k_to && k < asked;
            left[j] = there ? a.seg[(place(k) * ns + n) * a.width + e] : 0.0f;
            sum[j] = there ? a.sum[place(k) * a.width + e] : 0.0f;
        }
    };
    // The factor as two numbers: as one it may pass the range where its product with a small state does not (a rate above zero), or be
    // zero where an infinite state stays infinite token by token.  (12 x 1000 x 640 x 16 fp32: 13.5 us, with one number 12.5 us; looking
    // for such factors first, and with branches for them, it took as long.)
    auto next = [&](float h, float s, float l) __attribute__((always_inline)) {
        const float p = s * A2, part = __builtin_amdgcn_fmed3f(p, -126.0f, 126.0f), rest = __builtin_amdgcn_fmed3f(p - part, -126.0f, 128.0f);
        return s < 0.0f || h == 0.0f ? l : __builtin_fmaf(exp2_(part), h * exp2_(rest), l);
    };
    float h = first;
    if constexpr (J > 1) {
        float total = 0;
        h = 0;
        for (int k0 = k_from; k0 < k_to; k0 += M) {
            read(k0);
#pragma unroll
            for (int j = 0; j < M; j++) h = next(h, sum[j], left[j]), total = total < 0.0f || sum[j] < 0.0f ? -1.0f : total + sum[j];
        }
        meet[0][mine][c] = h, meet[1][mine][c] = total;
        __syncthreads();
        h = first;
        for (int k = 0; k < mine; k++) h = next(h, meet[1][k][c], meet[0][k][c]);
    }
    if (!on) return;
    for (int k0 = k_from; k0 < k_to; k0 += M) {
        if (J == 1 || per > M) read(k0);
#pragma unroll
        for (int j = 0; j < M; j++)
            if (k0 + j < k_to) {
                a.seg[(place(k0 + j) * ns + n) * a.width + e] = h;
                h = next(h, sum[j], left[j]);
            }
    }
    if (backward && a.dstate != nullptr && real && k_to == last + 1 && k_from <= last)
        a.dstate[(b * a.width + e) * a.states + n] = end > 0 ? h : first;         // a row without tokens leaves what came in
}

// ---- sums of M values over the 64 lanes of a wave: every step adds one half of the lanes to the other and halves the values that
// a lane carries, so that M values take about 2 M instructions.  Lane l gets the sum of value l / (64 / M). ----
template <int CTRL, int COUNT> __device__ __forceinline__ void fold(float *v, bool high) {      // COUNT values to COUNT / 2, or one value over both halves
    if constexpr (COUNT == 1) v[0] += dpp<CTRL>(v[0]);
    else {
#pragma unroll
        for (int k = 0; k < COUNT / 2; k++) {
            float keep = high ? v[k + COUNT / 2] : v[k], give = high ? v[k] : v[k + COUNT / 2];
            v[k] = keep + dpp<CTRL>(give);
        }
    }
}
__device__ __forceinline__ float first_sum(float x, float y) {      // the first step: value k and value k + M / 2
    swap32(x, y);
    return x + y;
}
template <int M> __device__ __forceinline__ float wave_sums(float (&v)[M / 2]) {
    static_assert(M >= 8 && M <= 64 && (M & (M - 1)) == 0, "a power of two");
    int lane = threadIdx.x % kWave;
#pragma unroll
    for (int k = 0; k < M / 4; k++) {
        swap16(v[k], v[k + M / 4]);
        v[k] += v[k + M / 4];
    }
    fold<kRor8, M / 4>(v, lane & 8);
    fold<kHalfMirror, (M / 8 > 1 ? M / 8 : 1)>(v, lane & 4);
    fold<kQuad2, (M / 16 > 1 ? M / 16 : 1)>(v, lane & 2);
    fold<kQuad1, (M / 32 > 1 ? M / 32 : 1)>(v, lane & 1);
    return v[0];
}

// The backward pass walks over a segment from its end, kept state by kept state.  From one it goes forward over kKept tokens with what
// each of them keeps of the state before it, a_t h_{t-1}, in registers, and then backward over them.  dB and dC are summed over the
// wave's channels token by token (wave_sums), over the block's waves after kKept tokens, over blocks by scan_bc_out.  Tokens past the
// row's end count with d = u = dy = 0, which leaves g as it is and adds nothing.
// More than 16 states are two halves (H = 2), each a wave's: what a token's gradients need of both, its output and two sums over the
// states, meets in shared memory, and each of the two waves finishes every second token (405 x 66 x 874 x 32 bf16 with the forward
// pass 1120 us when it was built; 4413 us without it where all states are one wave's, most of that for registers that do not fit).
// Bound by the vector unit: 2048 x 64 x 512 x 16 bf16 take some 1.0 ms, 403 instructions (466 issue slots) a token and wave, 98 of them for
// the way there, at 84 % of the slots with the two waves to a SIMD that the registers allow: all 256, and 8 more in 28 bytes of scratch.  Three waves with half the tokens each, whose registers spill within them, took a quarter longer.
template <class T, int NS, int H, bool PAD> __global__ __launch_bounds__(256, 2) void scan_backward(ScanArgs a) {
    using raw = typename T::raw;
    constexpr int SUB = kKept, M = 2 * NS, ALL = NS * H;
    extern __shared__ float pool[];
    const int lane = threadIdx.x % kWave, wave = uniform(threadIdx.x / kWave), waves = blockDim.x / kWave, half = H > 1 ? wave % H : 0, first_n = half * NS;
    const int lanes = blockDim.x / H, mine = wave / H * kWave + lane;            // the block's channels, and the lane's among them
    float *sums = pool;                                                          // [2][waves][SUB][M]
    float *meet = pool + 2 * waves * SUB * M;                                    // H > 1: [2][waves][SUB][3][64]
    int part = blockIdx.x % a.across, group = blockIdx.x / a.across, turn = 0;
    float dA[NS], dD = 0, dbias = 0, A2[NS];
    {
        int at = part * lanes + mine;
        rates<NS>(a, at < a.width ? at : a.width - 1, A2, first_n);
    }
#pragma unroll
    for (int n = 0; n < NS; n++) dA[n] = 0;
    for (int64_t item = group; item < a.batch * a.segments; item += a.groups) {
        Place p(*fresh_args(), item, part, lanes, mine);
        int64_t stop = p.t1 < p.end ? p.t1 : p.end;
        bool whole_end = p.end <= p.t1 && (p.end > p.t0 || p.seg == 0);
        const uint32_t bytes = p.bytes(sizeof(raw));
        if (p.t0 < stop || whole_end) {
            float g[NS];
            if (a.segments > 1) get_row<NS>(a.seg, p.b * a.segments + p.seg, a, p.e, g, ALL, first_n);
            else first_state<NS>(a.dlast, a, p.b, p.e, g, first_n);
            if (!p.on)
#pragma unroll
                for (int n = 0; n < NS; n++) g[n] = 0;
            float D = a.D != nullptr ? a.D[p.e] : 0.0f, bias = a.dt_bias != nullptr ? a.dt_bias[p.e] : 0.0f;

            // tokens t .. t + SUB - 1, `here` of which are the row's; bit i of `begins`: an episode begins at token t + i
            auto walk = [&](int64_t t, int here, uint32_t begins, float (&h)[NS]) __attribute__((always_inline)) {
                float keep[SUB][NS], d[SUB];
                raw ru[SUB], rd[SUB], early[4];
                FixedArgs *in = fresh_args();
                Line<raw> lu((const raw *)in->u, p.b * in->u_batch + t * in->u_time, in->u_time), ld((const raw *)in->dt, p.b * in->dt_batch + t * in->dt_time, in->dt_time),
                    ly((const raw *)in->dy, p.b * in->dy_batch + t * in->dy_time, in->dy_time), lz((const raw *)in->z, p.b * in->z_batch + t * in->z_time, in->z_time);
                const bool gated = in->z != nullptr;
                int states = in->states;
#pragma unroll
                for (int q = 0; q < SUB; q++) {
                    int at = q < here ? q : here - 1;
                    ru[q] = lu.get(bytes, at), rd[q] = ld.get(bytes, at);
                }
                early[0] = ld.get(bytes, here - 1), early[1] = ly.get(bytes, here - 1), early[2] = lz.get(bytes, here - 1), early[3] = lu.get(bytes, here - 1);
                Fixed *bc = fixed(in->bc + (p.b * in->length + t) * 2 * ALL + first_n);
                constexpr int S = NS / 2;
                One<NS> B[2];
                Pair<S> m, m2;
                auto token = [&](int q) __attribute__((always_inline)) { return bc + (q < here ? q : here - 1) * 2 * ALL; };
                B[0].read(token(0));
                uint32_t unseen = begins | ~0u << here;          // where no state is seen from: nothing behind the row sees its last one, which may be infinite
#pragma unroll
                for (int q = 0; q < SUB; q++) {
                    B[q & 1].hold();
                    asm volatile("" : "+s"(bc), "+s"(here), "+s"(unseen));         // no comparison held for later, no B kept for the way back
                    if (q + 1 < SUB) B[~q & 1].read(token(q + 1));
                    else m.read(token(q), ALL);
                    here_only();
                    d[q] = q < here ? softplus_(up<T>(rd[q]) + bias) : 0.0f;
                    float x = q < here ? d[q] * up<T>(ru[q]) : 0.0f;
                    if (unseen >> q & 1) forget<NS>(h);
#pragma unroll
                    for (int n = 0; n < NS; n++) {
                        keep[q][n] = exp2_(d[q] * A2[n]) * h[n];
                        h[n] = __builtin_fmaf(x, B[q & 1].v[n], keep[q][n]);
                        if (n % 4 == 3)
#pragma unroll
                            for (int k = n - 3; k <= n; k++) asm volatile("" : "+v"(keep[q][k]), "+v"(h[k]));
                    }
                    here_only();
                }
                // from here on the compiler does not know d: it would rather keep every exp and state of the walk before (2 x SUB x NS
                // registers more) than take them again
#pragma unroll
                for (int q = 0; q < SUB; q++) asm volatile("" : "+v"(d[q]));
                float *to = sums + (turn * waves + wave) * SUB * M;
                float *others = meet + (turn * waves + wave) * SUB * 3 * kWave + lane;
                FixedArgs *out_to = fresh_args();
                const int64_t row = (p.b * out_to->length + t) * out_to->width;
                Line<raw> gu((raw *)out_to->du, row, out_to->width), gd((raw *)out_to->ddt, row, out_to->width), gz((raw *)out_to->dz, row, out_to->width);
                // a token's gradients from its sums over all states.  Without branches: where one path stores and the other does not, the
                // wait for the next token's inputs would be one for the stores as well (without z the last store goes nowhere; 1427 us
                // with the forward pass, 1450 us with a branch).
                auto finish = [&](int q, float out, float zf, float sig, float o, float y, float gB, float gk, float raw_d, float dq, float uq) __attribute__((always_inline)) {
                    float dd = __builtin_fmaf(uq, gB, gk * kLn2), draw = q < here ? dd * sigmoid_(raw_d) : 0.0f;
                    const uint32_t where = q < here ? bytes : kOutside;
                    dD = __builtin_fmaf(o, uq, dD);
                    dbias += draw;
                    gu.put(down<T>(__builtin_fmaf(D, o, dq * gB)), where, q);
                    gd.put(down<T>(draw), where, q);
                    gz.put(down<T>(out * __builtin_fmaf(D, uq, y) * sig * (1.0f + zf * (1.0f - sig))), where, q);
                };
#pragma unroll
                for (int q = SUB - 1; q >= 0; q--) {
                    asm volatile("" : "+s"(here), "+s"(begins));
                    if (PAD) asm volatile("" : "+s"(states));
                    m.hold();
                    m2.read(token(q) + S, ALL);
                    here_only();
                    float raw_d = up<T>(early[0]) + bias, out = q < here ? up<T>(early[1]) : 0.0f, uq = q < here ? up<T>(early[3]) : 0.0f, zf = 0, gate = 1, sig = 0;
                    if (gated) {
                        zf = up<T>(early[2]);
                        sig = sigmoid_(zf);
                        gate = zf * sig;
                    }
                    if (q > 0) {                 // the token before, one token ahead
                        int at = q - 1 < here ? q - 1 : here - 1;
                        early[0] = ld.get(bytes, at), early[1] = ly.get(bytes, at), early[2] = lz.get(bytes, at), early[3] = lu.get(bytes, at);
                    }
                    float o = out * gate, x = d[q] * uq, gB = 0, gk = 0, y = 0, v[NS];
#pragma unroll
                    for (int n0 = 0; n0 < NS; n0 += 4) {
                        auto second_half = [&]() __attribute__((always_inline)) {
                            here_only();
                            m2.hold();
                            if (q > 0) m.read(token(q - 1), ALL);
                            here_only();
                        };
                        if (n0 == S) second_half();
                        // four states at a time, their sums added up here and not when they are next asked for: what the compiler
                        // would keep for later does not fit the registers.  some: those behind the first may be padding
                        auto four = [&](bool some) __attribute__((always_inline)) {
#pragma unroll
                            for (int k = n0; k < n0 + 4; k++) asm volatile("" : "+v"(keep[q][k]), "+v"(g[k]));
#pragma unroll
                            for (int n = n0; n < n0 + 4; n++) {
                                if (n == S && n != n0) second_half();
                                const float Bn = n < S ? m.B[n % S] : m2.B[n % S], Cn = n < S ? m.C[n % S] : m2.C[n % S];
                                float hn = __builtin_fmaf(x, Bn, keep[q][n]);
                                g[n] = __builtin_fmaf(o, Cn, g[n]);
                                v[n] = first_sum(g[n] * x, o * hn);
                                float gh = g[n] * keep[q][n];
                                if (!some || n == n0 || first_n + n < states) {
                                    y = __builtin_fmaf(Cn, hn, y);
                                    gB = __builtin_fmaf(g[n], Bn, gB);
                                    gk = __builtin_fmaf(gh, A2[n], gk);
                                    if (some && n > n0) asm volatile("" : "+v"(y), "+v"(gB), "+v"(gk));
                                }
                                dA[n] = __builtin_fmaf(gh, d[q], dA[n]);
                                g[n] *= exp2_(d[q] * A2[n]);
                            }
#pragma unroll
                            for (int k = n0; k < n0 + 4; k++) asm volatile("" : "+v"(dA[k]), "+v"(g[k]), "+v"(v[k]));
                        };
                        if (!PAD || (H == 1 && n0 + 4 <= fewest_states<NS>())) four(false);
                        else if (first_n + n0 < states) four(true);
                        else {
#pragma unroll
                            for (int k = n0; k < n0 + 4; k++) v[k] = 0;
                        }
                    }
                    if (begins >> q & 1) forget<NS>(g);
                    if constexpr (H == 1) {
                        finish(q, out, zf, sig, o, y, gB, gk, raw_d, d[q], uq);
                    } else others[(q * 3 + 0) * kWave] = y, others[(q * 3 + 1) * kWave] = gB, others[(q * 3 + 2) * kWave] = gk;
                    float total = wave_sums<M>(v);
                    if (lane % (kWave / M) == 0) to[q * M + lane / (kWave / M)] = total;
                    here_only();
                }
                // the other half of `sums` and `meet` is read by nobody after this barrier, and this half is written again after the next
                __syncthreads();
                if constexpr (H > 1) {
                    const float *both = meet + (turn * waves + wave / H * H) * SUB * 3 * kWave + lane;
                    for (int q = half; q < here; q += H) {
                        float uq = up<T>(lu.get(bytes, q)), raw_d = up<T>(ld.get(bytes, q)) + bias, out = up<T>(ly.get(bytes, q)), zf = 0, gate = 1, sig = 0, s[3] = {0, 0, 0};
                        if (gated) {
                            zf = up<T>(lz.get(bytes, q));
                            sig = sigmoid_(zf);
                            gate = zf * sig;
                        }
#pragma unroll
                        for (int k = 0; k < 3; k++)
#pragma unroll
                            for (int w = 0; w < H; w++) s[k] += both[((w * SUB + q) * 3 + k) * kWave];
                        finish(q, out, zf, sig, out * gate, s[0], s[1], s[2], raw_d, softplus_(raw_d), uq);
                    }
                }
                const float *from = sums + turn * waves * SUB * M;
                FixedArgs *sums_to = fresh_args();
                float *bc_to = sums_to->part_bc + (((int64_t)part * sums_to->batch + p.b) * sums_to->length + t) * 2 * ALL;
                for (int k = threadIdx.x; k < here * 2 * ALL; k += blockDim.x) {
                    const int q = k / (2 * ALL), n = k % NS, of = k / NS % H, which = k / ALL % 2;       // [token][B | C][half][state]
                    float v = 0;
                    for (int w = of; w < waves; w += H) v += from[(w * SUB + q) * M + which * NS + n];
                    bc_to[k] = v;
                }
                turn ^= 1;
            };

            if (p.t0 < stop)
                for (int64_t c0 = p.t0 + (stop - 1 - p.t0) / kGroup * kGroup; c0 >= p.t0; c0 -= kGroup) {
                    uint32_t begins = group_mask(*fresh_args(), p.b, c0, p.end);
                    int count = (int)(c0 + kGroup < stop ? kGroup : stop - c0);
                    for (int i = (count - 1) / SUB * SUB; i >= 0; i -= SUB) {
                        float h[NS];
                        FixedArgs *states_of = fresh_args();
                        kept_row<NS>(*states_of, p.b * states_of->chunks + (c0 + i) / SUB, p.bytes(4), h, ALL, first_n);
                        walk(c0 + i, count - i < SUB ? count - i : SUB, begins >> i, h);
                    }
                }
            if (p.on && p.seg == 0 && a.segments == 1 && a.dstate != nullptr) last_state<NS>(a.dstate, a, p.b, p.e, g, first_n);
        }
        raw *du = (raw *)a.du + p.b * a.length * a.width, *ddt = (raw *)a.ddt + p.b * a.length * a.width, *dz = a.z != nullptr ? (raw *)a.dz + p.b * a.length * a.width : nullptr;
        if (p.on && half == 0)
            for (int64_t t = p.t0 > p.end ? p.t0 : p.end; t < p.t1; t++) {
                (du + t * a.width)[p.e] = (ddt + t * a.width)[p.e] = down<T>(0.0f);
                if (dz != nullptr) (dz + t * a.width)[p.e] = down<T>(0.0f);
            }
    }
    // dD and ddt_bias: each half has its tokens' part
    float other[2] = {0, 0};
    if constexpr (H > 1) {
        __syncthreads();
        sums[(wave * 2 + 0) * kWave + lane] = dD, sums[(wave * 2 + 1) * kWave + lane] = dbias;
        __syncthreads();
#pragma unroll
        for (int w = 1; w < H; w++)
#pragma unroll
            for (int k = 0; k < 2; k++)
                if (half == 0) other[k] += sums[((wave + w) * 2 + k) * kWave + lane];
    }
    int at = part * lanes + mine;
    if (at < a.width) {
        float *to = a.part + (int64_t)group * (ALL + 2) * a.width + at;
#pragma unroll
        for (int n = 0; n < NS; n++) to[(int64_t)(first_n + n) * a.width] = dA[n];
        if (half == 0) {
            to[(int64_t)ALL * a.width] = dD + other[0];
            to[(int64_t)(ALL + 1) * a.width] = dbias + other[1];
        }
    }
}

// four values to a thread
template <class T> __global__ __launch_bounds__(256) void scan_bc_out(const float *part, const int32_t *lengths, void *dB, void *dC, int64_t batch, int64_t length, int parts, int states,
                                                                       int ns) {
    using raw = typename T::raw;
    int64_t at = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4, all = batch * length * 2 * ns;
    if (at >= all) return;
    int n = (int)(at % ns);
    if (n >= states) return;
    int64_t rest = at / ns, token = rest >> 1;
    Vec<F32, 4> v = {};
    if (lengths == nullptr || token % length < row_length(lengths, token / length, length))
        for (int k = 0; k < parts; k++) {
            Vec<F32, 4> p = load<F32, 4>(part + k * all + at);
#pragma unroll
            for (int i = 0; i < 4; i++) v.v[i] += p.v[i];
        }
    Vec<T, 4> r;
#pragma unroll
    for (int i = 0; i < 4; i++) r.v[i] = down<T>(v.v[i]);
    store_some<T, 4>((raw *)(rest & 1 ? dC : dB) + token * states + n, r, states - n);
}

struct ScanOut {
    float *dA, *dD, *dbias;
    int width, states, ns;
    __device__ void operator()(int64_t col, float v) const {
        int n = (int)(col / width), e = (int)(col % width);
        if (n < states) {
            if (dA != nullptr) dA[(int64_t)e * states + n] = v;
        } else if (n == ns) {
            if (dD != nullptr) dD[e] = v;
        } else if (n == ns + 1 && dbias != nullptr) dbias[e] = v;
    }
};

// ---- one token ----
// Q lanes share a channel, four states each: the state goes through registers in 16-byte pieces, in order of memory.  Bound by memory:
// 8 bytes a state (4096 x 1024 x 16 bf16 in 114 us, 5.0 TB/s).  Q = 0, for all numbers of states but 4, 8, 16 and 32: a lane takes a channel's
// states one by one, bound by their round trips and scattered accesses (4096 x 1024 bf16 with 7 states 92 us, 12: 255 us, 24: 1380 us).
// A lane keeps its channel's parameters for up to kStepRows rows; a row's state is under way while the one before is worked on.
constexpr int kStepRows = 4;
template <class T, int Q> __global__ __launch_bounds__(256) void scan_step(ScanArgs a, const void *B, const void *C, int64_t B_batch, int64_t C_batch, int64_t each) {
    using raw = typename T::raw;
    constexpr int kLanesOf = Q > 0 ? Q : 1, W = Q > 0 ? 4 : 1;
    int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x, row = at / kLanesOf;
    if (row >= each * a.width) return;               // whole groups of Q lanes leave together
    int q = (int)(at % kLanesOf), e = (int)(row % a.width);
    int64_t b0 = row / a.width;                      // rows b0, b0 + each, ..
    float bias = a.dt_bias != nullptr ? a.dt_bias[e] : 0.0f, D = a.D != nullptr ? a.D[e] : 0.0f;
    const float *A = a.A + (int64_t)e * a.states;
    Vec<F32, W> A2, next, h;
    if constexpr (Q > 0) {
        A2 = load<F32, W>(A + q * 4);
#pragma unroll
        for (int i = 0; i < W; i++) A2.v[i] *= kLog2e;
    }
    raw next_u = 0, next_dt = 0, next_z = 0;
    auto fetch = [&](int64_t b) __attribute__((always_inline)) {
        next_u = ((const raw *)a.u)[b * a.u_batch + e], next_dt = ((const raw *)a.dt)[b * a.dt_batch + e];
        if (a.z != nullptr) next_z = ((const raw *)a.z)[b * a.z_batch + e];
        if constexpr (Q > 0) next = load<F32, W>(a.state + (b * a.width + e) * a.states + q * 4);
    };
    fetch(b0);
    for (int64_t b = b0; b < a.batch; b += each) {
        float uf = up<T>(next_u), d = softplus_(up<T>(next_dt) + bias), zf = up<T>(next_z), x = d * uf, o = 0;
        h = next;
        if (b + each < a.batch) fetch(b + each);
        bool first = a.reset != nullptr && a.reset[b * a.reset_batch] != 0;
        const raw *Bp = (const raw *)B + b * B_batch, *Cp = (const raw *)C + b * C_batch;
        float *to = a.last + (b * a.width + e) * a.states;
        if constexpr (Q > 0) {
            Vec<T, W> Bv = load<T, W>(Bp + q * 4), Cv = load<T, W>(Cp + q * 4);
#pragma unroll
            for (int i = 0; i < W; i++) {
                float keep = first ? 0.0f : exp2_(d * A2.v[i]) * h.v[i];
                h.v[i] = __builtin_fmaf(x, up<T>(Bv.v[i]), keep);
                o = __builtin_fmaf(up<T>(Cv.v[i]), h.v[i], o);
            }
            store<F32, W>(to + q * 4, h);
            o = lane_sum<Q>(o);
        } else {
            const float *from = a.state + (b * a.width + e) * a.states;
            for (int n = 0; n < a.states; n++) {
                float keep = first ? 0.0f : exp2_(d * (A[n] * kLog2e)) * from[n];
                float hn = __builtin_fmaf(x, up<T>(Bp[n]), keep);
                o = __builtin_fmaf(up<T>(Cp[n]), hn, o);
                to[n] = hn;
            }
        }
        if (q == 0) {
            o = __builtin_fmaf(D, uf, o);
            if (a.z != nullptr) o *= zf * sigmoid_(zf);
            ((raw *)a.y)[b * a.width + e] = down<T>(o);
        }
    }
}

// ---- host ----
// The states that a lane walks with.  Powers of two where a backward pass follows, whose sums over a wave halve them step by step;
// 12 and 24 too where none does (3 x 5000 x 777 x 12 fp16 110 us, padded to 16 states 125 us).
static int scan_ns(const mws_scan_args *a, bool backward) {
    int n = a->states;
    if (!backward && a->kept == nullptr && n > 8) return n <= 12 ? 12 : n <= 16 ? 16 : n <= 24 ? 24 : 32;
    return n <= 4 ? 4 : n <= 8 ? 8 : n <= 16 ? 16 : 32;
}

struct ScanPlan {
    int ns, lanes, across, segments, span, groups;
    int64_t chunks;
    int64_t bc, seg, sum, part_bc, part, bytes;      // offsets into the workspace, in floats
};

// Waves of a block: as many as leave none of them without channels.
static int block_waves(int waves, int most) {
    int best = 1;
    for (int w = 2; w <= most; w++)
        if (waves % w == 0) best = w;
    return best;
}

// Segments: how many times kKept tokens each.  kKept tokens of one wave alone take a SIMD 3 us forward and 10.5 us backward, for what
// its instructions wait for; several waves take their issue slots' time (49 + 6 ns and 110 + 22 ns slots a token, four cycles each)
// and some of that once.  Each wave begins with its rates and state.  Cutting costs a second walk (0.8 of the first, backward 0.25),
// two launches and a step of scan_join for each segment.  (3 x 5000 x 777 x 12 fp16 forward, full rows, in segments of 8 tokens 171 us, of
// 24: 122, of 40: 112, of 48, which this takes: 109, of 64: 107, of 128: 137 us; 1 x 300 x 512 x 16 bf16 of 8, which this takes: 22, of
// 32: 39, of 64: 59 us.)
static int64_t best_span(int64_t waves, int64_t parts, int ns, bool backward) {
    const double alone = backward ? 10.5 : 3, slots = backward ? 110 + 22 * ns : 49 + 6 * ns, busy = slots * kKept * 4 / 2400, walks = backward ? 1.25 : 1.8;
    auto time = [&](int64_t w, int64_t each) {
        double one = alone * (double)each + 1.5, all = ((double)ceil_div(w, kSimds) + 0.7) * (busy * (double)each + (backward ? 0.08 : 0.04) * ns);
        return one > all ? one : all;
    };
    int64_t best = parts;
    double least = time(waves, parts);
    for (int64_t each = 1; each < parts; each = each < 16 ? each + 1 : each + each / 8) {
        int64_t count = ceil_div(parts, each);
        if (count > 1024) continue;
        double cost = time(waves * count, each) * walks + 5 + 0.08 * (double)count;
        if (cost < least) best = each, least = cost;
    }
    return best;
}

static ScanPlan scan_plan(const mws_scan_args *a, bool backward) {
    ScanPlan p = {};
    p.ns = scan_ns(a, backward);
    int waves = (int)ceil_div(a->width, kWave), of_block = block_waves(waves, lanes_of(p.ns) / kWave);
    p.lanes = of_block * kWave;
    p.across = (int)ceil_div(a->width, p.lanes);
    p.chunks = ceil_div(a->length, kKept);
    // (a forward pass is cut alike whether a backward pass follows or not: the same values to the last bit)
    int64_t parts = ceil_div(a->length > 0 ? a->length : 1, kKept), halves = backward && p.ns > 16 ? 2 : 1, each = best_span(a->batch * p.across * of_block * halves, parts, halves == 2 ? 16 : scan_ns(a, true), backward);
    p.segments = (int)ceil_div(parts, each);
    p.span = (int)(each * kKept);
    // blocks over the items, four rounds of the places at most: each leaves partial sums of dA, dD and ddt_bias
    int64_t items = a->batch * p.segments, most = 8 * kSimds / (of_block * halves * p.across) > 0 ? 8 * kSimds / (of_block * halves * p.across) : 1;
    p.groups = (int)(items < most ? items : most);
    int64_t at = 0, tokens = a->batch * a->length;
    auto take = [&at](int64_t n) {
        int64_t from = at;
        at += (n + 63) / 64 * 64;
        return from;
    };
    p.bc = take((tokens + 1) * 2 * p.ns);            // and what is asked for behind the last token
    p.seg = take(p.segments > 1 ? a->batch * p.segments * p.ns * a->width : 0);
    p.sum = take(p.segments > 1 ? a->batch * p.segments * a->width : 0);
    p.part_bc = take(backward ? p.across * tokens * 2 * p.ns : 0);
    p.part = take(backward ? (int64_t)p.groups * (p.ns + 2) * a->width : 0);
    p.bytes = at * (int64_t)sizeof(float);
    return p;
}

static int32_t scan_check(const mws_scan_args *a, const char *what, bool backward, bool step, bool pointers) {
    if (a == nullptr) return fail("%s: no arguments", what);
    if (a->type < MWS_F32 || a->type > MWS_F16) return fail("%s: type %d is none of MWS_F32, MWS_BF16, MWS_F16", what, a->type);
    if (a->states < 1 || a->states > MWS_SCAN_MAX_STATES) return fail("%s: %d states are not within 1 .. %d", what, a->states, MWS_SCAN_MAX_STATES);
    if (a->width < 1 || a->width > (1 << 22)) return fail("%s: width %d", what, a->width);
    if (a->batch < 0 || a->length < 0 || a->batch > (1 << 30) || a->length > (1 << 30) || a->batch * (a->length + 1) > ((int64_t)1 << 33)) return fail("%s: %lld rows of %lld tokens", what, (long long)a->batch, (long long)a->length);
    if (step && a->length != 1) return fail("%s: one token at a time", what);
    for (int64_t stride : {a->u_time, a->dt_time, a->z_time, a->dy_time})
        if (stride < 0 || stride > MWS_SCAN_MAX_STRIDE) return fail("%s: tokens %lld values apart", what, (long long)stride);
    if (!pointers) return 0;
    if (a->A == nullptr) return fail("%s: A is NULL", what);
    if (a->batch == 0) return 0;
    if (a->length > 0 && (a->u == nullptr || a->dt == nullptr || a->B == nullptr || a->C == nullptr)) return fail("%s: u, dt, B or C is NULL", what);
    if (!backward && a->length > 0 && a->y == nullptr) return fail("%s: y is NULL", what);
    if (backward && a->length > 0 && (a->dy == nullptr || a->kept == nullptr || a->du == nullptr || a->ddt == nullptr || a->dB == nullptr || a->dC == nullptr)) return fail("%s: dy, kept, du, ddt, dB or dC is NULL", what);
    if (backward && a->length > 0 && a->z != nullptr && a->dz == nullptr) return fail("%s: dz is NULL", what);
    if (step && (a->state == nullptr || a->last == nullptr)) return fail("%s: the state is NULL", what);
    return 0;
}

static ScanArgs scan_device(const mws_scan_args *a, const ScanPlan &p) {
    ScanArgs d = {};
    float *w = (float *)a->workspace;
    d.u = a->u, d.dt = a->dt, d.z = a->z, d.dy = a->dy, d.A = a->A, d.D = a->D, d.dt_bias = a->dt_bias, d.state = a->state, d.dlast = a->dlast;
    d.reset = a->reset, d.lengths = a->lengths, d.y = a->y, d.du = a->du, d.ddt = a->ddt, d.dz = a->z != nullptr ? a->dz : nullptr;
    d.last = a->last, d.kept = a->kept, d.dstate = a->dstate;
    if (w != nullptr) d.bc = w + p.bc, d.seg = w + p.seg, d.sum = w + p.sum, d.part_bc = w + p.part_bc, d.part = w + p.part;
    d.batch = a->batch, d.length = a->length, d.chunks = p.chunks;
    d.u_batch = a->u_batch, d.u_time = a->u_time, d.dt_batch = a->dt_batch, d.dt_time = a->dt_time, d.z_batch = a->z_batch, d.z_time = a->z_time;
    d.dy_batch = a->dy_batch, d.dy_time = a->dy_time, d.reset_batch = a->reset_batch, d.reset_time = a->reset_time;
    d.width = a->width, d.states = a->states, d.across = p.across, d.segments = p.segments, d.span = p.span, d.groups = p.groups;
    return d;
}

template <class T, int NS> static void spread_go(const mws_scan_args *a, const ScanArgs &d, hipStream_t stream) {
    if (a->batch * a->length > 0)
        hipLaunchKernelGGL((spread<T, NS>), dim3((unsigned)ceil_div(a->length * (2 * NS / 4), 256), (unsigned)(a->batch < 32768 ? a->batch : 32768)), dim3(256), 0, stream, a->B, a->C,
                           const_cast<float *>(d.bc), a->batch, a->length, a->B_batch, a->B_time, a->C_batch, a->C_time, a->states);
}
static void join_go(const ScanArgs &d, int ns, bool backward, hipStream_t stream) {
    const int j = joiners(d.batch * d.states * d.width, d.segments);
    dim3 grid((unsigned)ceil_div(d.batch * ns * d.width, 256 / j));
    if (j == 8) hipLaunchKernelGGL(scan_join<8>, grid, dim3(256), 0, stream, d, ns, backward);
    else if (j == 4) hipLaunchKernelGGL(scan_join<4>, grid, dim3(256), 0, stream, d, ns, backward);
    else hipLaunchKernelGGL(scan_join<1>, grid, dim3(256), 0, stream, d, ns, backward);
}

template <class T, int NS, bool PAD> static void forward_go(const mws_scan_args *a, const ScanPlan &p, const ScanArgs &d, hipStream_t stream) {
    spread_go<T, NS>(a, d, stream);
    dim3 grid((unsigned)(d.batch * p.segments * p.across)), block(p.lanes);
    if (p.segments > 1) {
        hipLaunchKernelGGL((scan_segment<T, NS>), grid, block, 0, stream, d);
        join_go(d, NS, false, stream);
    }
    hipLaunchKernelGGL((scan_forward<T, NS, PAD>), grid, block, 0, stream, d);
}
template <class T, int NS, bool PAD> static void backward_go(const mws_scan_args *a, const ScanPlan &p, const ScanArgs &d, hipStream_t stream) {
    constexpr int H = NS > 16 ? 2 : 1, PER = NS / H;
    dim3 block(p.lanes);
    spread_go<T, NS>(a, d, stream);
    if (p.segments > 1 && d.batch > 0) {
        hipLaunchKernelGGL((scan_segment_back<T, NS>), dim3((unsigned)(d.batch * p.segments * p.across)), block, 0, stream, d);
        join_go(d, NS, true, stream);
    }
    // 14 KB a wave of a half, 56 KB for the four of a block; 8 KB for four waves without halves: under the 64 KB that a block has without
    // asking for more
    const int waves = p.lanes / kWave * H;
    size_t lds = (size_t)2 * waves * kKept * (2 * PER + (H > 1 ? 3 * kWave : 0)) * sizeof(float);
    if (d.batch > 0) hipLaunchKernelGGL((scan_backward<T, PER, H, PAD>), dim3((unsigned)(p.groups * p.across)), dim3(waves * kWave), lds, stream, d);
    int64_t count = d.batch * d.length * 2 * NS;
    if (count > 0)
        hipLaunchKernelGGL((scan_bc_out<T>), dim3((unsigned)ceil_div(count / 4, 256)), dim3(256), 0, stream, d.part_bc, a->lengths, a->dB, a->dC, d.batch, d.length, p.across, a->states, NS);
    ScanOut out = {a->dA, a->dD, a->ddt_bias, a->width, a->states, NS};
    launch_sum_parts(d.part, p.groups, (int64_t)(NS + 2) * a->width, out, stream);
}
template <class T, bool PAD> static void scan_go(const mws_scan_args *a, const ScanPlan &p, const ScanArgs &d, bool backward, hipStream_t stream) {
#define MWS_GO(NS) (backward ? backward_go<T, NS, PAD>(a, p, d, stream) : forward_go<T, NS, PAD>(a, p, d, stream))
    if (p.ns == 4) MWS_GO(4);
    else if (p.ns == 8) MWS_GO(8);
    else if (p.ns == 12) forward_go<T, 12, PAD>(a, p, d, stream);
    else if (p.ns == 16) MWS_GO(16);
    else if (p.ns == 24) forward_go<T, 24, PAD>(a, p, d, stream);
    else MWS_GO(32);
#undef MWS_GO
}
template <class T> static void scan_type(const mws_scan_args *a, const ScanPlan &p, const ScanArgs &d, bool backward, hipStream_t stream) {
    if (a->states == p.ns) scan_go<T, false>(a, p, d, backward, stream);
    else scan_go<T, true>(a, p, d, backward, stream);
}
static void scan_run(const mws_scan_args *a, const ScanPlan &p, const ScanArgs &d, bool backward, hipStream_t stream) {
    if (a->type == MWS_F32) scan_type<F32>(a, p, d, backward, stream);
    else if (a->type == MWS_BF16) scan_type<BF16>(a, p, d, backward, stream);
    else scan_type<F16>(a, p, d, backward, stream);
}
static int step_lanes_of(const mws_scan_args *a) { return a->states == 4 ? 1 : a->states == 8 ? 2 : a->states == 16 ? 4 : a->states == 32 ? 8 : 0; }
static int64_t step_rows(const mws_scan_args *a, int64_t &lanes) {
    int q = step_lanes_of(a);
    lanes = (int64_t)a->width * (q > 0 ? q : 1);
    return step_lanes(a->batch, lanes, kStepRows);
}
static int64_t step_blocks(const mws_scan_args *a) {
    int64_t lanes, each = step_rows(a, lanes);
    return ceil_div(each * lanes, 256);
}
template <class T> static void step_go(const mws_scan_args *a, const ScanArgs &d, hipStream_t stream) {
    int q = step_lanes_of(a);
    int64_t lanes, each = step_rows(a, lanes);
    dim3 grid((unsigned)ceil_div(each * lanes, 256));
#define MWS_GO(Q) hipLaunchKernelGGL((scan_step<T, Q>), grid, dim3(256), 0, stream, d, a->B, a->C, a->B_batch, a->C_batch, each)
    if (q == 1) MWS_GO(1);
    else if (q == 2) MWS_GO(2);
    else if (q == 4) MWS_GO(4);
    else if (q == 8) MWS_GO(8);
    else MWS_GO(0);
#undef MWS_GO
}
}  // namespace mws

using namespace mws;

extern "C" int64_t mws_scan_kept(const mws_scan_args *a) {
    if (int32_t e = scan_check(a, "mws_scan_kept", false, false, false)) return e;
    return a->batch * ceil_div(a->length, kKept) * scan_ns(a, true) * a->width;
}

extern "C" int64_t mws_scan_workspace(const mws_scan_args *a, int32_t backward) {
    if (int32_t e = scan_check(a, "mws_scan_workspace", false, false, false)) return e;
    return scan_plan(a, backward != 0).bytes;
}

// whether the launches can count their threads.  dB's and dC's kernel counts its values, four times its threads.
static bool scan_fits(const mws_scan_args *a, const ScanPlan &p, bool backward) {
    return fits(a->batch * p.segments * p.across, p.lanes) && (!backward || fits(ceil_div(a->batch * a->length * 2 * p.ns, 256), 256)) && fits(ceil_div(a->length * 2 * p.ns / 4, 256), 256) &&
           (p.segments <= 1 || fits(ceil_div(a->batch * p.ns * a->width, 256), 256)) && fits(ceil_div((int64_t)(p.ns + 2) * a->width, 32), 1024);
}

static int32_t scan_call(const mws_scan_args *a, const char *what, bool backward, void *stream) {
    if (int32_t e = scan_check(a, what, backward, false, true)) return e;
    ScanPlan p = scan_plan(a, backward);
    if (a->workspace_bytes < p.bytes || (p.bytes > 0 && a->workspace == nullptr)) return fail("%s: the workspace needs %lld bytes", what, (long long)p.bytes);
    if (!backward && a->batch == 0) return 0;
    // (a pass that is recorded, before its backward pass would be refused)
    if (!scan_fits(a, p, backward) || (!backward && a->kept != nullptr && !scan_fits(a, scan_plan(a, true), true)))
        return fail("%s: %lld rows of %lld tokens, %d channels and %d states are more than one launch can count", what, (long long)a->batch, (long long)a->length, a->width, a->states);
    scan_run(a, p, scan_device(a, p), backward, (hipStream_t)stream);
    return launched(what);
}
extern "C" int32_t mws_scan_forward(const mws_scan_args *a, void *stream) { return scan_call(a, "mws_scan_forward", false, stream); }
extern "C" int32_t mws_scan_backward(const mws_scan_args *a, void *stream) { return scan_call(a, "mws_scan_backward", true, stream); }

extern "C" int32_t mws_scan_step(const mws_scan_args *a, void *stream) {
    if (int32_t e = scan_check(a, "mws_scan_step", false, true, true)) return e;
    if (a->batch == 0) return 0;
    if (!fits(step_blocks(a), 256)) return fail("mws_scan_step: %lld rows of %d channels are more than one launch can count", (long long)a->batch, a->width);
    ScanPlan none = {};
    ScanArgs d = scan_device(a, none);
    if (a->type == MWS_F32) step_go<F32>(a, d, (hipStream_t)stream);
    else if (a->type == MWS_BF16) step_go<BF16>(a, d, (hipStream_t)stream);
    else step_go<F16>(a, d, (hipStream_t)stream);
    return launched("mws_scan_step");
}
