/*
 * mwseq.h -- C ABI of libmwseq.so: the operators of a policy with memory on the device (layer norm, the short causal
 * convolution, the selective state space scan), forward, backward and for one token.
 *
 * Conventions: every function checks its arguments on the host, launches on `stream` (a hipStream_t; NULL: the default stream) of
 * the CURRENT device, does not wait, and returns 0 or a negative code; the message is available through mws_last_error() (one per
 * thread).  All pointers but the argument struct are device pointers owned by the caller.  The library holds no state and no
 * device memory: scratch memory is the caller's `workspace`, of at least the bytes that the _workspace function returns for the
 * same struct (pointers in it are looked at for being NULL or not, nothing else); two calls that may run at the same time need
 * workspaces of their own.  Pointers are aligned as their elements are, workspaces as float.
 *
 * Activations are MWS_F32, MWS_BF16 or MWS_F16 (`type`); their last dimension is contiguous, the strides of the others are given
 * in elements.  Parameters are float or of the activations' type (`param_type`).  Sums, statistics and scan states are float.
 *
 * Tokens are [batch, length].  `reset` (uint8 [batch, length] by strides, may be NULL): non-zero where an episode begins, so that
 * neither the state nor any earlier token of the row is seen from there on.  `lengths` (int32 [batch], may be NULL): how many
 * tokens of a row count, taken into [0, length]; outputs and gradients of the others are zero, their inputs are not used.
 *
 * Sizes of which one launch would need 2^32 threads or more (2^26 rows of one token) are refused, and scans with 2^32 values of dB and
 * dC together (2^27 tokens of 16 states), both backward and forward with `kept`.
 */
#ifndef MWSEQ_H
#define MWSEQ_H
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

enum { MWS_F32 = 0, MWS_BF16 = 1, MWS_F16 = 2 };
enum { MWS_ARGUMENT = -1, MWS_LAUNCH = -2 };

#define MWS_NORM_MAX_WIDTH 16384
#define MWS_CONV_MIN_TAPS 2
#define MWS_CONV_MAX_TAPS 4
#define MWS_SCAN_MAX_STATES 32
#define MWS_SCAN_MAX_STRIDE (1 << 26)   /* from one token to the next of u, dt, z and dy, in values */

/* y = (x - mean) / sqrt(var + eps) * weight + bias over rows of `width`; weight and bias may be NULL */
typedef struct mws_norm_args {
    const void *x, *weight, *bias, *dy;   /* [rows, width]; [width]; [width]; [rows, width] (backward) */
    void *y, *dx, *dweight, *dbias;       /* contiguous; y: forward; the others: backward, each may be NULL */
    void *workspace;
    int64_t rows, x_stride, dy_stride;
    int64_t workspace_bytes;
    int32_t width, type, param_type;
    float eps;
} mws_norm_args;

/* y_t = silu(bias + sum_j weight[:, j] x_{t - taps + 1 + j}); the inputs before the first token come from `state` (NULL: zeros) */
typedef struct mws_conv_args {
    const void *x, *weight, *bias, *state, *dy, *dlast;   /* [B, T, E]; [E, taps]; [E]; [B, taps - 1, E]; [B, T, E]; as state */
    const uint8_t *reset;
    const int32_t *lengths;
    void *y, *last;                            /* contiguous; last: the state after the row's last token (step: may be `state` itself) */
    void *dx, *dweight, *dbias, *dstate;       /* contiguous, backward, each may be NULL (dlast NULL: zeros) */
    void *workspace;
    int64_t batch, length;
    int64_t x_batch, x_time, dy_batch, dy_time, reset_batch, reset_time;
    int64_t workspace_bytes;
    int32_t width, taps, type, param_type;
} mws_conv_args;

/* d_t = softplus(dt_t + dt_bias), h_t = exp(d_t A) h_{t-1} + d_t B_t u_t, y_t = (sum_n C_t h_t + D u_t) silu(z_t);
 * h_{-1} is `state` (NULL: zeros); D, z and dt_bias may be NULL */
typedef struct mws_scan_args {
    const void *u, *dt, *z, *B, *C, *dy;       /* [batch, length, width], B and C [batch, length, states] */
    const float *A, *D, *dt_bias, *state, *dlast;   /* [width, states]; [width]; [width]; [batch, width, states]; as state */
    const uint8_t *reset;
    const int32_t *lengths;
    void *y;                                   /* contiguous, as every output */
    float *last;                               /* the state after the row's last token (step: may be `state` itself) */
    float *kept;                               /* forward, may be NULL: states for the backward pass, mws_scan_kept() floats; backward: the same */
    void *du, *ddt, *dz, *dB, *dC;             /* backward: of the activations' type; dz where z is */
    float *dA, *dD, *ddt_bias, *dstate;        /* backward: dD, ddt_bias and dstate where their inputs are */
    void *workspace;
    int64_t batch, length;
    int64_t u_batch, u_time, dt_batch, dt_time, z_batch, z_time, B_batch, B_time, C_batch, C_time, dy_batch, dy_time, reset_batch, reset_time;
    int64_t workspace_bytes;
    int32_t width, states, type, reserved;
} mws_scan_args;

const char *mws_last_error(void);
int64_t mws_sizeof(int32_t which);             /* 0, 1, 2: the size of mws_norm_args, mws_conv_args, mws_scan_args */

int32_t mws_norm_forward(const mws_norm_args *a, void *stream);
int64_t mws_norm_workspace(const mws_norm_args *a);            /* of the backward pass, in bytes; negative: an error */
int32_t mws_norm_backward(const mws_norm_args *a, void *stream);

int32_t mws_conv_forward(const mws_conv_args *a, void *stream);
int64_t mws_conv_workspace(const mws_conv_args *a);            /* of the backward pass */
int32_t mws_conv_backward(const mws_conv_args *a, void *stream);
int32_t mws_conv_step(const mws_conv_args *a, void *stream);   /* length 1; `last` gets the new state */

int64_t mws_scan_kept(const mws_scan_args *a);                 /* floats of `kept` */
int64_t mws_scan_workspace(const mws_scan_args *a, int32_t backward);
int32_t mws_scan_forward(const mws_scan_args *a, void *stream);
int32_t mws_scan_backward(const mws_scan_args *a, void *stream);
int32_t mws_scan_step(const mws_scan_args *a, void *stream);   /* length 1; `last` gets the new state */

#ifdef __cplusplus
}
#endif
#endif
