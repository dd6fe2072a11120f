// wnv_recurrence.hip -- the gated linear recurrence: a scan over (B, T, C), its backward pass, and one step with the state in place.
//
//   z = (f | v | o) along the channels,  u = 1 - sigmoid(f)
//   h_t = sigmoid(f_t) h_{t-1} + (1 - sigmoid(f_t)) v_t = h_{t-1} + u_t (v_t - h_{t-1})          y_t = h_t sigmoid(o_t)   (no o: y = h)
//
// The second form of h_t is what runs: a gate that remembers long has sigmoid(f) next to 1, where 32 bits leave it 6e-8 off, and a
// state that sums over 1 / u steps then is 6e-8 / u off; u itself is held to its own precision.
// h_{t-1} reads as zero at a step that begins an utterance of a packed slot (seg_start[b][t] == t).  Behind lengths[b] the state is
// handed on, y and the gradients are zero, and z is not looked at.
#include <hip/hip_runtime.h>

#include "wnv_hostutil.h"
#include "wnv_num.h"

namespace {

struct RecArgs {
    int B, C, gates;
    long long T, zb, zt;            // batch and time stride of z, in elements
    long long h0b;
    const void* z;
    const float* h0;
    const int *lengths, *seg_start;
    void* y;
    float* h_last;
    float* saved;                   // (B, T, C) states, for the backward pass
    const void* dy;
    long long dyb, dyt;
    const float* dh_last;
    void* dz;
    float* dh0;
};

constexpr int RT = 64;

template <typename E>
__global__ void __launch_bounds__(RT) wnv_recurrence_fwd(RecArgs a) {
    const int c = blockIdx.x * RT + threadIdx.x, b = blockIdx.y;
    if (c >= a.C) return;
    const E* z = (const E*)a.z + (long long)b * a.zb + c;
    E* y = (E*)a.y + (long long)b * a.T * a.C + c;
    const long long n = a.lengths ? min((long long)a.lengths[b], a.T) : a.T;
    float h = a.h0 ? a.h0[(long long)b * a.h0b + c] : 0.f;
    for (long long t = 0; t < a.T; ++t) {
        float out = 0.f;
        if (t < n) {
            float keep, u;
            wnv_gate(wnv_up(z[t * a.zt]), keep, u);
            if (a.seg_start && a.seg_start[(long long)b * a.T + t] == t) h = 0.f;
            h = fmaf(u, wnv_up(z[t * a.zt + a.C]) - h, h);
            out = h;
            if (a.gates == 3) {
                float so, uo;
                wnv_gate(wnv_up(z[t * a.zt + 2 * a.C]), so, uo);
                out = h * so;
            }
        }
        y[t * a.C] = wnv_down<E>(out);
        if (a.saved) a.saved[((long long)b * a.T + t) * a.C + c] = h;
    }
    a.h_last[(long long)b * a.C + c] = h;
}

// g_t = dy_t sigmoid(o_t);  dh_t = g_t + (what step t+1 hands back);  hands back dh_t sigmoid(f_t), nothing over a beginning
// df = dh (h_{t-1} - v) sigmoid(f) u;  dv = dh u;  do = dy h sigmoid(o) (1 - sigmoid(o))
template <typename E>
__global__ void __launch_bounds__(RT) wnv_recurrence_bwd(RecArgs a) {
    const int c = blockIdx.x * RT + threadIdx.x, b = blockIdx.y;
    if (c >= a.C) return;
    const E* z = (const E*)a.z + (long long)b * a.zb + c;
    const E* dy = a.dy ? (const E*)a.dy + (long long)b * a.dyb + c : nullptr;
    E* dz = (E*)a.dz + (long long)b * a.T * a.gates * a.C + c;
    const float* hs = a.saved + (long long)b * a.T * a.C + c;
    const long long n = a.lengths ? min((long long)a.lengths[b], a.T) : a.T;
    float r = a.dh_last ? a.dh_last[(long long)b * a.C + c] : 0.f;
    const float h0 = a.h0 ? a.h0[(long long)b * a.h0b + c] : 0.f;
    for (long long t = a.T - 1; t >= 0; --t) {
        float df = 0.f, dv = 0.f, dgo = 0.f;
        if (t < n) {
            float keep, u;
            wnv_gate(wnv_up(z[t * a.zt]), keep, u);
            const bool begins = a.seg_start && a.seg_start[(long long)b * a.T + t] == t;
            const float before = begins ? 0.f : t ? hs[(t - 1) * a.C] : h0, v = wnv_up(z[t * a.zt + a.C]);
            float g = dy ? wnv_up(dy[t * a.dyt]) : 0.f;
            if (a.gates == 3) {
                float so, uo;
                wnv_gate(wnv_up(z[t * a.zt + 2 * a.C]), so, uo);
                dgo = g * hs[t * a.C] * so * uo;
                g *= so;
            }
            const float dh = g + r;
            df = dh * (before - v) * keep * u;
            dv = dh * u;
            r = begins ? 0.f : fmaf(-u, dh, dh);
        }
        E* d = dz + t * a.gates * a.C;
        d[0] = wnv_down<E>(df);
        d[a.C] = wnv_down<E>(dv);
        if (a.gates == 3) d[2 * a.C] = wnv_down<E>(dgo);
    }
    if (a.dh0) a.dh0[(long long)b * a.C + c] = r;
}

template <typename E>
__global__ void __launch_bounds__(RT) wnv_recurrence_one(const E* z, long long zb, float* state, E* y, int C, int gates) {
    const int c = blockIdx.x * RT + threadIdx.x, b = blockIdx.y;
    if (c >= C) return;
    z += (long long)b * zb + c;
    float keep, u, h = state[(long long)b * C + c];
    wnv_gate(wnv_up(z[0]), keep, u);
    h = fmaf(u, wnv_up(z[C]) - h, h);
    state[(long long)b * C + c] = h;
    if (gates == 3) {
        float so, uo;
        wnv_gate(wnv_up(z[2 * C]), so, uo);
        h *= so;
    }
    y[(long long)b * C + c] = wnv_down<E>(h);
}

#define WNV_BY_TYPE(dtype, ...)                                                       \
    switch (dtype) {                                                                  \
        case WNV_F32: { using E = float; __VA_ARGS__; break; }                        \
        case WNV_BF16: { using E = wnv_bf16; __VA_ARGS__; break; }                    \
        default: { using E = wnv_f16; __VA_ARGS__; break; }                           \
    }

wnv_status check_shape(const char* who, int device, int64_t B, int64_t T, int64_t C, int gates, int dtype) {
    if (device < 0) return fail(WNV_ERR_INVALID_ARG, "%s: device must be >= 0", who);
    if (B <= 0 || T <= 0 || C <= 0) return fail(WNV_ERR_INVALID_ARG, "%s: B, T and C must be positive", who);
    if (T > INT32_MAX) return fail(WNV_ERR_UNSUPPORTED, "%s: at most 2^31 - 1 steps", who);
    if (B > 65535 || C > (1 << 20)) return fail(WNV_ERR_UNSUPPORTED, "%s: at most 65535 rows and 2^20 channels", who);
    if (gates != 2 && gates != 3) return fail(WNV_ERR_INVALID_ARG, "%s: gates must be 2 (f, v) or 3 (f, v, o)", who);
    if (!wnv_dtype_size(dtype)) return fail(WNV_ERR_INVALID_ARG, "%s: unknown dtype %d", who, dtype);
    return WNV_OK;
}

wnv_status launched(const char* who) {
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? WNV_OK : fail(WNV_ERR_HIP, "%s: launch failed: %s", who, hipGetErrorString(e));
}

wnv_status check_strides(const char* who, const wnv_recurrence_args* a) {
    if (a->z_batch_stride < 0 || a->z_time_stride < 0 || (a->h0 && a->h0_batch_stride < 0) ||
        (a->dy && (a->dy_batch_stride < 0 || a->dy_time_stride < 0)))
        return fail(WNV_ERR_INVALID_ARG, "%s: negative stride", who);
    return WNV_OK;
}

RecArgs device_args(const wnv_recurrence_args* a) {
    RecArgs k{};
    k.B = a->B; k.C = a->C; k.gates = a->gates; k.T = a->T;
    k.zb = a->z_batch_stride; k.zt = a->z_time_stride; k.h0b = a->h0_batch_stride;
    k.z = a->z; k.h0 = a->h0; k.lengths = a->lengths; k.seg_start = a->seg_start;
    k.y = a->y; k.h_last = a->h_last; k.saved = (float*)a->saved;
    k.dy = a->dy; k.dyb = a->dy_batch_stride; k.dyt = a->dy_time_stride;
    k.dh_last = a->dh_last; k.dz = a->dz; k.dh0 = a->dh0;
    return k;
}

}  // namespace

extern "C" int64_t wnv_recurrence_saved_bytes(int32_t B, int64_t T, int32_t C, int32_t gates, int32_t dtype) {
    if (check_shape("wnv_recurrence_saved_bytes", 0, B, T, C, gates, dtype) != WNV_OK) return -1;
    return (int64_t)B * T * C * 4;
}

extern "C" int64_t wnv_recurrence_workspace_bytes(int32_t B, int64_t T, int32_t C, int32_t gates, int32_t dtype) {
    if (check_shape("wnv_recurrence_workspace_bytes", 0, B, T, C, gates, dtype) != WNV_OK) return -1;
    return 0;
}

extern "C" wnv_status wnv_recurrence_forward(int32_t device, const wnv_recurrence_args* a) {
    if (!a || !a->z || !a->y || !a->h_last) return fail(WNV_ERR_INVALID_ARG, "wnv_recurrence_forward: NULL argument");
    if (wnv_status st = check_shape("wnv_recurrence_forward", device, a->B, a->T, a->C, a->gates, a->dtype)) return st;
    if (wnv_status st = check_strides("wnv_recurrence_forward", a)) return st;
    DeviceGuard guard(device);
    if (!guard.ok) return fail(WNV_ERR_HIP, "wnv_recurrence_forward: cannot select device %d", device);
    const RecArgs k = device_args(a);
    const dim3 grid((a->C + RT - 1) / RT, a->B);
    WNV_BY_TYPE(a->dtype, hipLaunchKernelGGL(wnv_recurrence_fwd<E>, grid, dim3(RT), 0, (hipStream_t)a->stream, k));
    return launched("wnv_recurrence_forward");
}

extern "C" wnv_status wnv_recurrence_backward(int32_t device, const wnv_recurrence_args* a) {
    if (!a || !a->z || !a->saved || !a->dz) return fail(WNV_ERR_INVALID_ARG, "wnv_recurrence_backward: NULL argument");
    if (wnv_status st = check_shape("wnv_recurrence_backward", device, a->B, a->T, a->C, a->gates, a->dtype)) return st;
    if (wnv_status st = check_strides("wnv_recurrence_backward", a)) return st;
    DeviceGuard guard(device);
    if (!guard.ok) return fail(WNV_ERR_HIP, "wnv_recurrence_backward: cannot select device %d", device);
    const RecArgs k = device_args(a);
    const dim3 grid((a->C + RT - 1) / RT, a->B);
    WNV_BY_TYPE(a->dtype, hipLaunchKernelGGL(wnv_recurrence_bwd<E>, grid, dim3(RT), 0, (hipStream_t)a->stream, k));
    return launched("wnv_recurrence_backward");
}

extern "C" wnv_status wnv_recurrence_step(int32_t device, const void* z, int64_t z_batch_stride, float* state, void* y, int32_t B,
                                          int32_t C, int32_t gates, int32_t dtype, void* stream) {
    if (!z || !state || !y) return fail(WNV_ERR_INVALID_ARG, "wnv_recurrence_step: NULL argument");
    if (z_batch_stride < 0) return fail(WNV_ERR_INVALID_ARG, "wnv_recurrence_step: negative stride");
    if (wnv_status st = check_shape("wnv_recurrence_step", device, B, 1, C, gates, dtype)) return st;
    DeviceGuard guard(device);
    if (!guard.ok) return fail(WNV_ERR_HIP, "wnv_recurrence_step: cannot select device %d", device);
    const dim3 grid((C + RT - 1) / RT, B);
    WNV_BY_TYPE(dtype, hipLaunchKernelGGL(wnv_recurrence_one<E>, grid, dim3(RT), 0, (hipStream_t)stream, (const E*)z,
                                          (long long)z_batch_stride, state, (E*)y, C, gates));
    return launched("wnv_recurrence_step");
}
