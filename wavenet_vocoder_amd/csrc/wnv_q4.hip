// wnv_q4.hip -- products of a few rows with weights of 4 bits: y = x W^T + bias, W[n, k] = scale[n, k/g] (code[n, k] - zero[n, k/g]),
// and the step of the gated recurrence (wnv_recurrence.hip) straight behind the product with its gates.
//
// Weights are laid out once, in tiles of 16 rows x 128 inputs: lane l of a wave holds row l % 16 and, in word j of its 16 bytes, the
// inputs 32 j + 8 (l / 16) ... + 7 of the tile -- what a 16 x 16 x 32 matrix instruction wants of a lane.  Inputs 2p and 2p + 1 of a
// word sit at bits 4p and 16 + 4p.  The rows of each gate are padded to a multiple of 16, so that one tile of each gate holds the
// same channels; scales and zero points are stored [tile][group][16 rows], the bias [tile][16 rows].
#include <hip/hip_runtime.h>

#include "wnv_hostutil.h"
#include "wnv_num.h"

namespace {

struct Q4Dev {
    int cin, rows, gates, group;    // rows: of one gate
    int tiles, kb, groups;          // tiles of one gate, 128-wide blocks and groups along the inputs (padded)
    const uint4* codes;             // [gates * tiles][kb][64]
    const wnv_bf16* scales;         // [gates * tiles][groups][16]
    const uint8_t* zeros;           // [gates * tiles][groups][16]
    const float* bias;              // [gates * tiles][16]
};

__global__ void __launch_bounds__(256) wnv_q4_pack(const uint8_t* codes, const wnv_bf16* scales, const uint8_t* zeros, const float* bias,
                                                   Q4Dev q, int n_groups, uint32_t* pcodes, wnv_bf16* pscales, uint8_t* pzeros,
                                                   float* pbias, int* bad) {
    const long long words = (long long)q.gates * q.tiles * q.kb * 256, gs = (long long)q.gates * q.tiles * q.groups * 16;
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
    if (i < words) {
        const int j = i & 3, lane = (i >> 2) & 63;
        const long long tb = i >> 8;
        const int kb = tb % q.kb, tile = tb / q.kb;
        const int row = (tile % q.tiles) * 16 + lane % 16, k0 = kb * 128 + j * 32 + (lane / 16) * 8;
        uint32_t w = 0;
        if (row < q.rows) {
            const uint8_t* src = codes + ((long long)(tile / q.tiles) * q.rows + row) * q.cin;
            for (int e = 0; e < 8; ++e)
                if (k0 + e < q.cin) {
                    const uint32_t v = src[k0 + e];
                    if (v > 15) *bad = 1;
                    w |= (v & 15) << (4 * (e / 2) + 16 * (e & 1));
                }
        }
        pcodes[i] = w;
    }
    if (i < gs) {
        const int r = i & 15;
        const long long tg = i >> 4;
        const int g = tg % q.groups, tile = tg / q.groups, row = (tile % q.tiles) * 16 + r;
        wnv_bf16 s = (wnv_bf16)0.f;
        uint8_t zp = 0;
        if (row < q.rows && g < n_groups) {
            const long long src = ((long long)(tile / q.tiles) * q.rows + row) * n_groups + g;
            s = scales[src];
            zp = zeros ? zeros[src] : 8;
            if (zp > 15) *bad = 1;
        }
        pscales[i] = s;
        pzeros[i] = zp;
    }
    if (i < (long long)q.gates * q.tiles * 16) {
        const int tile = i >> 4, row = (tile % q.tiles) * 16 + (int)(i & 15);
        pbias[i] = bias && row < q.rows ? bias[(tile / q.tiles) * q.rows + row] : 0.f;
    }
}

// Asymmetric rounding of one group by one thread: the range is widened to hold zero, the scale is a 15th of it, rounded up to bf16 so
// that the codes still reach both ends; zero and codes go by the rounded scale.
__global__ void __launch_bounds__(256) wnv_q4_quantise(const float* w, int cout, int cin, int group, int n_groups, uint8_t* codes,
                                                       wnv_bf16* scales, uint8_t* zeros, int* bad) {
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
    if (i >= (long long)cout * n_groups) return;
    const int g = i % n_groups, k1 = min(cin, (g + 1) * group);
    const long long row = i / n_groups;
    float lo = 0.f, hi = 0.f;
    for (int k = g * group; k < k1; ++k) {
        const float v = w[row * cin + k];
        if (!(fabsf(v) <= 3.0e38f)) *bad = 1;
        lo = fminf(lo, v);
        hi = fmaxf(hi, v);
    }
    const float want = hi * (1.f / 15.f) - lo * (1.f / 15.f);
    wnv_bf16 sb = (wnv_bf16)want;
    if ((float)sb < want) sb = __builtin_bit_cast(wnv_bf16, (uint16_t)(__builtin_bit_cast(uint16_t, sb) + 1));
    const float s = (float)sb, zp = s > 0.f ? fminf(rintf(-lo / s), 15.f) : 0.f;
    scales[i] = sb;
    zeros[i] = (uint8_t)zp;
    for (int k = g * group; k < k1; ++k) {
        const float v = s > 0.f ? rintf(w[row * cin + k] / s) + zp : 0.f;
        codes[row * cin + k] = (uint8_t)fminf(fmaxf(v, 0.f), 15.f);
    }
}

__global__ void __launch_bounds__(256) wnv_q4_unpack(Q4Dev q, float* w) {
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
    if (i >= (long long)q.gates * q.rows * q.cin) return;
    const int k = i % q.cin;
    const long long n = i / q.cin;
    const int row = n % q.rows;
    const long long tile = (n / q.rows) * q.tiles + row / 16;
    const int lane = ((k >> 3) & 3) * 16 + row % 16, j = (k >> 5) & 3, e = k & 7;
    const uint32_t word = ((const uint32_t*)(q.codes + (tile * q.kb + k / 128) * 64 + lane))[j];
    const long long at = (tile * q.groups + k / q.group) * 16 + row % 16;
    w[i] = (float)q.scales[at] * ((float)((word >> (4 * (e / 2) + 16 * (e & 1))) & 15) - (float)q.zeros[at]);
}

struct Q4Call {
    const void* x;
    long long xs;                   // row stride of x, in elements
    void* y;
    float* state;                   // the recurrence step: (B, rows), in place; else null
    int B;
};

// One wave per tile of 16 channels and row of x, a lane per weight row and quarter of the inputs.
template <typename E, int GATES, bool STEP>
__global__ void __launch_bounds__(64) wnv_q4_rows(Q4Dev q, Q4Call a) {
    const int lane = threadIdx.x, r = lane % 16, quarter = lane / 16, b = blockIdx.y;
    const E* x = (const E*)a.x + b * a.xs;
    float z[GATES];
    for (int g = 0; g < GATES; ++g) {
        const long long tile = STEP ? (long long)g * q.tiles + blockIdx.x : blockIdx.x;
        float acc = 0.f;
        for (int kb = 0; kb < q.kb; ++kb) {
            const uint4 w = q.codes[(tile * q.kb + kb) * 64 + lane];
            const uint32_t words[4] = {w.x, w.y, w.z, w.w};
            for (int j = 0; j < 4; ++j) {
                const int k0 = kb * 128 + j * 32 + quarter * 8;
                const long long at = (tile * q.groups + k0 / q.group) * 16 + r;
                const float zero = (float)q.zeros[at];
                float sum = 0.f;
                for (int e = 0; e < 8; ++e)
                    if (k0 + e < q.cin)
                        sum = fmaf(wnv_up(x[k0 + e]), (float)((words[j] >> (4 * (e / 2) + 16 * (e & 1))) & 15) - zero, sum);
                acc = fmaf((float)q.scales[at], sum, acc);
            }
        }
        acc += __shfl_xor(acc, 16);
        acc += __shfl_xor(acc, 32);
        z[g] = acc + q.bias[tile * 16 + r];
    }
    if (quarter != 0) return;
    if (!STEP) {
        const int gate = blockIdx.x / q.tiles, row = (blockIdx.x % q.tiles) * 16 + r;
        if (row < q.rows) ((E*)a.y)[((long long)b * q.gates + gate) * q.rows + row] = wnv_down<E>(z[0]);
        return;
    }
    const int row = blockIdx.x * 16 + r;
    if (row >= q.rows) return;
    float h = a.state[(long long)b * q.rows + row];
    h = fmaf(wnv_gate(-z[0]), z[GATES > 1 ? 1 : 0] - h, h);
    a.state[(long long)b * q.rows + row] = h;
    if (GATES == 3) h *= wnv_gate(z[GATES > 2 ? 2 : 0]);
    ((E*)a.y)[(long long)b * q.rows + row] = wnv_down<E>(h);
}

#define WNV_BY_TYPE(dtype, ...)                                                       \
    switch (dtype) {                                                                  \
        case WNV_F32: { using E = float; __VA_ARGS__; break; }                        \
        case WNV_BF16: { using E = wnv_bf16; __VA_ARGS__; break; }                    \
        default: { using E = wnv_f16; __VA_ARGS__; break; }                           \
    }

struct Alloc {                      // a device buffer that goes with its scope
    void* p = nullptr;
    ~Alloc() { if (p) (void)hipFree(p); }
};

bool capturing(hipStream_t s) {
    hipStreamCaptureStatus st = hipStreamCaptureStatusNone;
    return hipStreamIsCapturing(s, &st) == hipSuccess && st != hipStreamCaptureStatusNone;
}

}  // namespace

struct wnv_q4 {
    Q4Dev q{};
    int device = 0;
    Scratch codes, scales, zeros, bias;
    bool loaded = false;
};

extern "C" wnv_status wnv_q4_create(int32_t cin, int32_t cout, int32_t gates, int32_t group, int32_t device, wnv_q4_handle* out) {
    if (!out) return fail(WNV_ERR_INVALID_ARG, "wnv_q4_create: out handle is NULL");
    *out = nullptr;
    if (device < 0) return fail(WNV_ERR_INVALID_ARG, "wnv_q4_create: device must be >= 0");
    if (cin <= 0 || cout <= 0 || gates < 1 || gates > 3 || cout % gates)
        return fail(WNV_ERR_INVALID_ARG, "wnv_q4_create: bad geometry (cin %d, cout %d, gates %d)", cin, cout, gates);
    if (group != 32 && group != 64 && group != 128)
        return fail(WNV_ERR_UNSUPPORTED, "wnv_q4_create: groups of %d inputs (32, 64 and 128 are implemented)", group);
    if (cin > (1 << 20) || cout > (1 << 20) || (int64_t)cin * cout > INT32_MAX)
        return fail(WNV_ERR_UNSUPPORTED, "wnv_q4_create: at most 2^20 inputs, 2^20 outputs and 2^31 - 1 weights");
    wnv_q4* h = new wnv_q4();
    h->device = device;
    Q4Dev& q = h->q;
    q.cin = cin; q.rows = cout / gates; q.gates = gates; q.group = group;
    q.tiles = (q.rows + 15) / 16; q.kb = (cin + 127) / 128; q.groups = q.kb * (128 / group);
    *out = h;
    return WNV_OK;
}

static wnv_status q4_pack(wnv_q4* h, const uint8_t* codes, const wnv_bf16* scales, const uint8_t* zeros, const float* bias, int* bad,
                          hipStream_t s) {
    Q4Dev& q = h->q;
    const size_t tiles = (size_t)q.gates * q.tiles, words = tiles * q.kb * 256, gs = tiles * q.groups * 16;
    h->loaded = false;
    HIP_TRY(h->codes.ensure(words * 4));
    HIP_TRY(h->scales.ensure(gs * 2));
    HIP_TRY(h->zeros.ensure(gs));
    HIP_TRY(h->bias.ensure(tiles * 64));
    q.codes = (const uint4*)h->codes.p; q.scales = (const wnv_bf16*)h->scales.p; q.zeros = (const uint8_t*)h->zeros.p;
    q.bias = (const float*)h->bias.p;
    hipLaunchKernelGGL(wnv_q4_pack, dim3((unsigned)((std::max(words, gs) + 255) / 256)), dim3(256), 0, s, codes, scales, zeros, bias, q,
                       (q.cin + q.group - 1) / q.group, (uint32_t*)h->codes.p, (wnv_bf16*)h->scales.p, (uint8_t*)h->zeros.p,
                       (float*)h->bias.p, bad);
    HIP_TRY(hipGetLastError());
    int found = 0;
    HIP_TRY(hipMemcpyAsync(&found, bad, sizeof found, hipMemcpyDeviceToHost, s));
    HIP_TRY(hipStreamSynchronize(s));
    if (found) return fail(WNV_ERR_INVALID_ARG, "wnv_q4: a code or zero point is over 15, or a weight is not finite");
    h->loaded = true;
    return WNV_OK;
}

extern "C" wnv_status wnv_q4_set_codes(wnv_q4_handle h, const uint8_t* codes, const void* scales, const uint8_t* zeros, const float* bias,
                                       void* stream) {
    if (!h || !codes || !scales) return fail(WNV_ERR_INVALID_ARG, "wnv_q4_set_codes: NULL argument");
    hipStream_t s = (hipStream_t)stream;
    DeviceGuard guard(h->device);
    if (!guard.ok) return fail(WNV_ERR_HIP, "wnv_q4_set_codes: cannot select device %d", h->device);
    if (capturing(s)) return fail(WNV_ERR_UNSUPPORTED, "wnv_q4_set_codes waits for the device: not while the stream is captured");
    Alloc bad;
    HIP_TRY(hipMalloc(&bad.p, 4));
    HIP_TRY(hipMemsetAsync(bad.p, 0, 4, s));
    return q4_pack(h, codes, (const wnv_bf16*)scales, zeros, bias, (int*)bad.p, s);
}

extern "C" wnv_status wnv_q4_set_weights(wnv_q4_handle h, const float* weight, const float* bias, void* stream) {
    if (!h || !weight) return fail(WNV_ERR_INVALID_ARG, "wnv_q4_set_weights: NULL argument");
    hipStream_t s = (hipStream_t)stream;
    DeviceGuard guard(h->device);
    if (!guard.ok) return fail(WNV_ERR_HIP, "wnv_q4_set_weights: cannot select device %d", h->device);
    if (capturing(s)) return fail(WNV_ERR_UNSUPPORTED, "wnv_q4_set_weights waits for the device: not while the stream is captured");
    const Q4Dev& q = h->q;
    const int cout = q.gates * q.rows, n_groups = (q.cin + q.group - 1) / q.group;
    const size_t gs = (size_t)cout * n_groups;
    Alloc codes, scales, zeros, bad;
    HIP_TRY(hipMalloc(&codes.p, (size_t)cout * q.cin));
    HIP_TRY(hipMalloc(&scales.p, gs * 2));
    HIP_TRY(hipMalloc(&zeros.p, gs));
    HIP_TRY(hipMalloc(&bad.p, 4));
    HIP_TRY(hipMemsetAsync(bad.p, 0, 4, s));
    hipLaunchKernelGGL(wnv_q4_quantise, dim3((unsigned)((gs + 255) / 256)), dim3(256), 0, s, weight, cout, q.cin, q.group, n_groups,
                       (uint8_t*)codes.p, (wnv_bf16*)scales.p, (uint8_t*)zeros.p, (int*)bad.p);
    HIP_TRY(hipGetLastError());
    return q4_pack(h, (uint8_t*)codes.p, (wnv_bf16*)scales.p, (uint8_t*)zeros.p, bias, (int*)bad.p, s);
}

extern "C" wnv_status wnv_q4_dequantise(wnv_q4_handle h, float* weight, void* stream) {
    if (!h || !weight) return fail(WNV_ERR_INVALID_ARG, "wnv_q4_dequantise: NULL argument");
    if (!h->loaded) return fail(WNV_ERR_NOT_LOADED, "wnv_q4: weights are not set");
    DeviceGuard guard(h->device);
    if (!guard.ok) return fail(WNV_ERR_HIP, "wnv_q4_dequantise: cannot select device %d", h->device);
    const size_t n = (size_t)h->q.gates * h->q.rows * h->q.cin;
    hipLaunchKernelGGL(wnv_q4_unpack, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, (hipStream_t)stream, h->q, weight);
    HIP_TRY(hipGetLastError());
    return WNV_OK;
}

static wnv_status q4_check(const char* who, wnv_q4_handle h, const void* x, int64_t xs, const void* y, int32_t B, int32_t dtype) {
    if (!h || !x || !y) return fail(WNV_ERR_INVALID_ARG, "%s: NULL argument", who);
    if (!h->loaded) return fail(WNV_ERR_NOT_LOADED, "%s: weights are not set", who);
    if (B <= 0 || xs < 0) return fail(WNV_ERR_INVALID_ARG, "%s: bad batch size or row stride", who);
    if (B > 65535) return fail(WNV_ERR_UNSUPPORTED, "%s: at most 65535 rows", who);
    if (!wnv_dtype_size(dtype)) return fail(WNV_ERR_INVALID_ARG, "%s: unknown dtype %d", who, dtype);
    return WNV_OK;
}

extern "C" wnv_status wnv_q4_step(wnv_q4_handle h, const void* x, int64_t x_row_stride, void* y, int32_t B, int32_t dtype, void* stream) {
    if (wnv_status st = q4_check("wnv_q4_step", h, x, x_row_stride, y, B, dtype)) return st;
    DeviceGuard guard(h->device);
    if (!guard.ok) return fail(WNV_ERR_HIP, "wnv_q4_step: cannot select device %d", h->device);
    const Q4Call a{x, x_row_stride, y, nullptr, B};
    const dim3 grid(h->q.gates * h->q.tiles, B);
    WNV_BY_TYPE(dtype, hipLaunchKernelGGL((wnv_q4_rows<E, 1, false>), grid, dim3(64), 0, (hipStream_t)stream, h->q, a));
    HIP_TRY(hipGetLastError());
    return WNV_OK;
}

extern "C" wnv_status wnv_q4_recurrence_step(wnv_q4_handle h, const void* x, int64_t x_row_stride, float* state, void* y, int32_t B,
                                             int32_t dtype, void* stream) {
    if (wnv_status st = q4_check("wnv_q4_recurrence_step", h, x, x_row_stride, y, B, dtype)) return st;
    if (!state) return fail(WNV_ERR_INVALID_ARG, "wnv_q4_recurrence_step: NULL argument");
    if (h->q.gates < 2) return fail(WNV_ERR_INVALID_ARG, "wnv_q4_recurrence_step: the handle was created with one gate (2: f, v; 3: f, v, o)");
    DeviceGuard guard(h->device);
    if (!guard.ok) return fail(WNV_ERR_HIP, "wnv_q4_recurrence_step: cannot select device %d", h->device);
    const Q4Call a{x, x_row_stride, y, state, B};
    const dim3 grid(h->q.tiles, B);
    if (h->q.gates == 3) {
        WNV_BY_TYPE(dtype, hipLaunchKernelGGL((wnv_q4_rows<E, 3, true>), grid, dim3(64), 0, (hipStream_t)stream, h->q, a));
    } else {
        WNV_BY_TYPE(dtype, hipLaunchKernelGGL((wnv_q4_rows<E, 2, true>), grid, dim3(64), 0, (hipStream_t)stream, h->q, a));
    }
    HIP_TRY(hipGetLastError());
    return WNV_OK;
}

extern "C" wnv_status wnv_q4_destroy(wnv_q4_handle h) {
    if (!h) return WNV_OK;
    DeviceGuard guard(h->device);
    h->codes.release();
    h->scales.release();
    h->zeros.release();
    h->bias.release();
    delete h;
    return WNV_OK;
}
