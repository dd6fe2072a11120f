// wnv_q4.hip -- products of a few rows with weights of 4 bits: y = x W^T + bias, W[n, k] = scale[n, k/g] (code[n, k] - zero[n, k/g]),
// and the step of the gated recurrence (wnv_recurrence.hip) straight behind the product with its gates.
//
// The matrix instruction does the dot products, with the weights as its rows and up to 16 rows of x as its columns, so that a code
// costs a shift and an and-or per pair, and not an operation per code and row of x: a 16-bit float 16 + code is a mask and a constant
// away from the code (f16: 0x4c00 | code << 6; bf16, times 2^-12: 0x3b80 | code << 3), exact, and a second instruction with -(16 + zero) in
// every place takes the offset out again: the sum of x (code - zero) over a group, in float32, which the group's scale then joins to the
// rest.  float32 x is cut into three bf16 parts that add up to it exactly; they share the weights.  (The 2^-12 is taken out at the end: 128
// products of up to 31 x stay below 2^12 x, which may be the type's largest number.)
//
// Weights are laid out once, in tiles of 16 rows x 128 inputs: lane l of a wave holds row l % 16 and, in word j of its 16 bytes, the
// inputs 32 j + 8 (l / 16) ... + 7 of the tile -- what a 16 x 16 x 32 matrix instruction wants of a lane.  Inputs 2p and 2p + 1 of a
// word sit at bits 4p and 16 + 4p.  The rows of each gate are padded to a multiple of 16, so that one tile of each gate holds the
// same channels.  Behind a tile's codes, in arrays of their own: its scales as [4 rows of a result lane][group], its zero points as
// [row][group], its bias.
#include <hip/hip_runtime.h>

#include "wnv_hostutil.h"
#include "wnv_num.h"

namespace {

struct Q4Dev {
    int cin, rows, gates, group;    // rows: of one gate
    int tiles, kb;                  // tiles of one gate, 128-wide blocks along the inputs
    int per_block;                  // groups in a block: 128 / group
    const uint4* codes;             // [gates * tiles][kb][64]
    const wnv_bf16* scales;         // [gates * tiles][kb][4][per_block][4]: row 4 a + b at [a][group][b]
    const uint8_t* zeros;           // [gates * tiles][kb][16][per_block]
    const float* bias;              // [gates * tiles][16]
};

__device__ __forceinline__ long long scale_at(const Q4Dev& q, long long tile, int group, int row) {
    return (((tile * q.kb + group / q.per_block) * 4 + row / 4) * q.per_block + group % q.per_block) * 4 + row % 4;
}
__device__ __forceinline__ long long zero_at(const Q4Dev& q, long long tile, int group, int row) {
    return ((tile * q.kb + group / q.per_block) * 16 + row) * q.per_block + group % q.per_block;
}

__global__ void __launch_bounds__(256) wnv_q4_pack(const uint8_t* codes, const wnv_bf16* scales, const uint8_t* zeros, const float* bias,
                                                   Q4Dev q, int n_groups, uint32_t* pcodes, wnv_bf16* pscales, uint8_t* pzeros,
                                                   float* pbias, int* bad) {
    const long long words = (long long)q.gates * q.tiles * q.kb * 256, gs = (long long)q.gates * q.tiles * q.kb * q.per_block * 16;
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
        const int groups = q.kb * q.per_block, g = tg % groups, tile = tg / groups, row = (tile % q.tiles) * 16 + r;
        wnv_bf16 s = (wnv_bf16)0.f;
        uint8_t zp = 0;
        if (row < q.rows && g < n_groups) {
            const long long src = ((long long)(tile / q.tiles) * q.rows + row) * n_groups + g;
            s = scales[src];
            zp = zeros ? zeros[src] : 8;
            if (zp > 15) *bad = 1;
        }
        pscales[scale_at(q, tile, g, r)] = s;
        pzeros[zero_at(q, tile, g, r)] = zp;
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
    const float code = (float)((word >> (4 * (e / 2) + 16 * (e & 1))) & 15), zero = (float)q.zeros[zero_at(q, tile, k / q.group, row % 16)];
    w[i] = (float)q.scales[scale_at(q, tile, k / q.group, row % 16)] * (code - zero);
}

struct Q4Call {
    const void* x;
    long long xs;                   // row stride of x, in elements
    void* y;
    float* state;                   // the recurrence step: (B, rows), in place; else null
    int B;
};

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef u32x4 u32x4_any __attribute__((aligned(1)));

// What the kernels need to know of x's type: the 16-bit float that its products run in, and how many parts of that make one x.
template <typename E> struct Q4Type;
template <> struct Q4Type<wnv_bf16> { static constexpr int PARTS = 1, AT = 3; static constexpr uint32_t ONE = 0x3b80u; static constexpr float UP = 4096.f; };
template <> struct Q4Type<wnv_f16> { static constexpr int PARTS = 1, AT = 6; static constexpr uint32_t ONE = 0x4c00u; static constexpr float UP = 1.f; };
template <> struct Q4Type<float> : Q4Type<wnv_bf16> { static constexpr int PARTS = 3; };

template <typename E> __device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
    if constexpr (__is_same(E, wnv_f16))
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// The 8 codes of a word as 16 + code (over UP), in the order of x's memory.
template <typename E> __device__ __forceinline__ u32x4 codes_up(uint32_t w) {
    constexpr int AT = Q4Type<E>::AT;
    constexpr uint32_t MASK = 0x000f000fu << AT, ONE = Q4Type<E>::ONE * 0x10001u;
    u32x4 r;
#pragma unroll
    for (int p = 0; p < 4; ++p) {
        const uint32_t s = 4 * p <= AT ? w << (AT - 4 * p) : w >> (4 * p - AT);
        r[p] = (s & MASK) | ONE;
    }
    return r;
}
template <typename E> __device__ __forceinline__ u32x4 offset_of(uint32_t zero) {        // -(16 + zero) (over UP), 8 times
    const uint32_t h = (zero << Q4Type<E>::AT) | Q4Type<E>::ONE | 0x8000u, w = h | h << 16;
    return u32x4{w, w, w, w};
}

// Eight inputs as they stand in memory, and cut into parts.
template <typename E> struct Inputs { u32x4 w[sizeof(E) / 2]; };
template <typename E> __device__ __forceinline__ Inputs<E> load_inputs(const E* p) {             // at any alignment
    Inputs<E> r;
#pragma unroll
    for (int i = 0; i < (int)sizeof(E) / 2; ++i) r.w[i] = *(const u32x4_any*)((const char*)p + 16 * i);
    return r;
}
template <typename E> __device__ __forceinline__ Inputs<E> load_inputs(const E* p, int left) {   // zeros behind the row's end
    if (left >= 8) return load_inputs(p);
    E e[8] = {};
#pragma unroll
    for (int i = 0; i < 7; ++i)
        if (i < left) e[i] = p[i];
    Inputs<E> r;
    __builtin_memcpy(&r, e, sizeof r);
    return r;
}
template <typename E> __device__ __forceinline__ void parts_of(const Inputs<E>& x, u32x4 (&part)[Q4Type<E>::PARTS]) {
    if constexpr (sizeof(E) == 2) {
        part[0] = x.w[0];
    } else {                            // the upper 8 bits of the 24, of what is left, and of what is left then: nothing remains
#pragma unroll
        for (int p = 0; p < 4; ++p) {
            const uint32_t w0 = x.w[p / 2][p % 2 * 2], w1 = x.w[p / 2][p % 2 * 2 + 1];
            const float r0 = __uint_as_float(w0) - __uint_as_float(w0 & 0xffff0000u), r1 = __uint_as_float(w1) - __uint_as_float(w1 & 0xffff0000u);
            const uint32_t m0 = __float_as_uint(r0), m1 = __float_as_uint(r1);
            const float s0 = r0 - __uint_as_float(m0 & 0xffff0000u), s1 = r1 - __uint_as_float(m1 & 0xffff0000u);
            part[0][p] = __builtin_amdgcn_perm(w1, w0, 0x07060302u);
            part[1][p] = __builtin_amdgcn_perm(m1, m0, 0x07060302u);
            part[2][p] = __builtin_amdgcn_perm(__float_as_uint(s1), __float_as_uint(s0), 0x07060302u);
        }
    }
}

// What a wave reads of the weights for one block of 128 inputs.
template <int GROUPS> struct Q4Block {
    uint4 code;
    uint2 scale[GROUPS];
    uint32_t zero;
};
template <int GROUPS> __device__ __forceinline__ Q4Block<GROUPS> load_block(const Q4Dev& q, long long at, int lane) {
    Q4Block<GROUPS> f;
    f.code = q.codes[at * 64 + lane];
    const uint2* s = (const uint2*)(q.scales + (at * 4 + lane / 16) * GROUPS * 4);
#pragma unroll
    for (int g = 0; g < GROUPS; ++g) f.scale[g] = s[g];
    const uint8_t* z = q.zeros + (at * 16 + lane % 16) * GROUPS;
    f.zero = GROUPS == 4 ? *(const uint32_t*)z : GROUPS == 2 ? *(const uint16_t*)z : *z;
    return f;
}

// NT tiles side by side (GATES > 0: one tile of each gate, of the same 16 channels, and the sums go straight into the recurrence's
// step) x 16 rows of x.  The blocks of 128 inputs are dealt to `split` slices, the slices to the `waves` waves of the same tiles (a
// gate's); the slices' sums are joined in LDS in their order: no atomics, and a row's result does not depend on the rows beside it
// (the split goes by the weights' shape alone).
// STAGED: the rows of x go through LDS behind the first weights' request, and the parts of float32 rows are columns of their own there
// (up to 5 rows); else each wave takes its own of x from L2, and the parts follow each other into sums of their own.  Both add the
// parts' sums in the same order at the end: which of the two runs does not show in the result.  The weights of a wave's next block are
// asked for before this one's products where registers allow it (STAGED).
template <typename E, int NT, int GROUPS, int GATES, bool STAGED>
__global__ void __launch_bounds__(NT == 1 ? 1024 : 512) wnv_q4_rows(Q4Dev q, Q4Call a, int split, int waves, int most) {
    static_assert(!GATES || NT == 1, "a wave holds one gate");
    extern __shared__ u32x4 shared[];   // STAGED: [part][row][16 kb + 1], 8 inputs each; then sums [gate][slice][NT][SUMS][64]
    constexpr int PARTS = Q4Type<E>::PARTS, SUMS = STAGED ? 1 : PARTS, JG = 4 / GROUPS;
    const int lane = threadIdx.x % 64, wave = threadIdx.x / 64, r = lane % 16, quarter = lane / 16;
    const int all = q.gates * q.tiles, tile0 = blockIdx.x * NT + (GATES ? wave / waves * q.tiles : 0), b0 = blockIdx.y * most;
    const int rows = min(most, a.B - b0), pitch = 16 * q.kb + 1;          // a pitch of 16 bytes more spreads the rows over the banks
    const E* x = (const E*)a.x + (long long)(b0 + min(r, rows - 1)) * a.xs;

    Q4Block<GROUPS> f[NT] = {};
    if (STAGED) {                       // one slice a wave: its first weights are on their way while x is staged
#pragma unroll
        for (int t = 0; t < NT; ++t) f[t] = load_block<GROUPS>(q, (long long)min(tile0 + t, all - 1) * q.kb + wave % waves, lane);
        for (int i = threadIdx.x; i < rows * 16 * q.kb; i += blockDim.x) {
            const int row = i / (16 * q.kb), k = i - row * (16 * q.kb);
            u32x4 part[PARTS];
            parts_of<E>(load_inputs<E>((const E*)a.x + (long long)(b0 + row) * a.xs + k * 8, q.cin - k * 8), part);
#pragma unroll
            for (int p = 0; p < PARTS; ++p) shared[(p * rows + row) * pitch + k] = part[p];
        }
        __syncthreads();
    }
    f32x4* sums = (f32x4*)shared + (STAGED ? PARTS * rows * pitch : 0);
    for (int slice = wave % waves; slice < split; slice += waves) {
        f32x4 acc[NT][SUMS] = {};
        for (int kb = slice; kb < q.kb; kb += split) {
            if (!STAGED) {
#pragma unroll
                for (int t = 0; t < NT; ++t) f[t] = load_block<GROUPS>(q, (long long)min(tile0 + t, all - 1) * q.kb + kb, lane);
            }
            Q4Block<GROUPS> next[NT] = {};
#pragma unroll
            for (int t = 0; t < NT; ++t)
                if (STAGED && kb + split < q.kb) next[t] = load_block<GROUPS>(q, (long long)min(tile0 + t, all - 1) * q.kb + kb + split, lane);
            Inputs<E> in[4] = {};
            if (!STAGED) {
                if ((kb + 1) * 128 <= q.cin) {
                    if (r < rows) {
#pragma unroll
                        for (int j = 0; j < 4; ++j) in[j] = load_inputs<E>(x + kb * 128 + j * 32 + quarter * 8);
                    }
                } else if (r < rows) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) in[j] = load_inputs<E>(x + kb * 128 + j * 32 + quarter * 8, q.cin - (kb * 128 + j * 32 + quarter * 8));
                }
            }
#pragma unroll
            for (int g = 0; g < GROUPS; ++g) {
                f32x4 sum[NT][SUMS] = {};
#pragma unroll
                for (int j = g * JG; j < (g + 1) * JG; ++j) {
                    u32x4 part[SUMS] = {};
                    if constexpr (!STAGED) parts_of<E>(in[j], part);
                    else if (r < PARTS * rows) part[0] = shared[r * pitch + kb * 16 + j * 4 + quarter];
#pragma unroll
                    for (int t = 0; t < NT; ++t) {
                        const u32x4 w = codes_up<E>(j == 0 ? f[t].code.x : j == 1 ? f[t].code.y : j == 2 ? f[t].code.z : f[t].code.w);
                        const u32x4 o = offset_of<E>(f[t].zero >> (8 * g) & 255);
#pragma unroll
                        for (int p = 0; p < SUMS; ++p) {
                            sum[t][p] = mfma<E>(w, part[p], sum[t][p]);
                            sum[t][p] = mfma<E>(o, part[p], sum[t][p]);
                        }
                    }
                }
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    const uint2 s = f[t].scale[g];
                    const f32x4 scale{__uint_as_float(s.x << 16), __uint_as_float(s.x & 0xffff0000u), __uint_as_float(s.y << 16),
                                      __uint_as_float(s.y & 0xffff0000u)};
#pragma unroll
                    for (int p = 0; p < SUMS; ++p)
#pragma unroll
                        for (int i = 0; i < 4; ++i) acc[t][p][i] = fmaf(scale[i], sum[t][p][i], acc[t][p][i]);
                }
            }
            if (STAGED) {
#pragma unroll
                for (int t = 0; t < NT; ++t) f[t] = next[t];
            }
        }
        f32x4* sum = sums + (long long)(wave / waves * split + slice) * (NT * SUMS * 64) + lane;
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int p = 0; p < SUMS; ++p) sum[(t * SUMS + p) * 64] = acc[t][p];
    }
    __syncthreads();

    // 16 neighbouring threads write 16 neighbouring outputs of a row; lane l of a result holds its column l % 16, rows 4 (l / 16) ...
    const float* part = (const float*)sums;
    for (int e = threadIdx.x; e < NT * 256; e += blockDim.x) {
        const int n = e % 16, col = e / 16 % 16, row = b0 + col, t = e / 256, tile = blockIdx.x * NT + t, gate = GATES ? 0 : tile / q.tiles;
        const int channel = (tile - gate * q.tiles) * 16 + n, at = (t * SUMS * 64 + n / 4 * 16 + col) * 4 + n % 4;
        const int apart = STAGED ? rows * 4 : 256;      // from a part's sum to the next one's
        if (col >= rows || tile >= all || channel >= q.rows) continue;
        float z[GATES ? GATES : 1];
#pragma unroll
        for (int g = 0; g < (GATES ? GATES : 1); ++g) {
            float sum = 0.f;
            for (int w = 0; w < split; ++w) {
                const float* one = part + at + (g * split + w) * (NT * SUMS * 256);
                sum += PARTS == 3 ? one[0] + one[apart] + one[2 * apart] : one[0];
            }
            z[g] = fmaf(sum, Q4Type<E>::UP, q.bias[(tile + g * q.tiles) * 16 + n]);
        }
        if (!GATES) {
            ((E*)a.y)[((long long)row * q.gates + gate) * q.rows + channel] = wnv_down<E>(z[0]);
        } else {
            float h = a.state[(long long)row * q.rows + channel];
            h = wnv_blend(z[0], h, z[GATES > 1 ? 1 : 0]);
            a.state[(long long)row * q.rows + channel] = h;
            if (GATES == 3) h *= wnv_gate(z[GATES - 1]);
            ((E*)a.y)[(long long)row * q.rows + channel] = wnv_down<E>(h);
        }
    }
}

#define WNV_BY_TYPE(dtype, ...)                                                       \
    switch (dtype) {                                                                  \
        case WNV_F32: { using E = float; __VA_ARGS__; break; }                        \
        case WNV_BF16: { using E = wnv_bf16; __VA_ARGS__; break; }                    \
        default: { using E = wnv_f16; __VA_ARGS__; break; }                           \
    }

// Which form runs (us a launch in a graph, both sides measured):
//  * x through LDS if its rows fit (two workgroups a CU then) and it pays: float32, whose three parts become columns of one product
//    (1 x 8192 x 8192: 11.6, from L2 23.4; 8 x 512 x 3 512 with the step: 4.4 and 5.4) -- at most 5 rows a workgroup, so that many rows
//    read the weights more often: as long as that is no more than two workgroups a CU (through LDS and from L2, 512 of them: 5 x 2048 x 8192
//    6.7 and 7.4, 16 x 2048 x 2048 6.7 and 7.2; more: 6 x 2048 x 8192 9.9 and 7.5, 64 x 2048 x 2048 17.5 and 9.1, 64 x 512 x 8192 16.8 and
//    9.7), and with the step always (24 x 2048 x 3 2048 13.6 and 16.1, 64 x 2048 x 3 2048 27.7 and 28.6) --, and 16-bit types if a wave
//    has several blocks of inputs to wait for (1 x 8192 x 8192 bf16: 11.1 and 13.2; 8 x 1616 x 512, one block a wave: 4.6 and 3.9).
//  * else two tiles a wave, which halves what is read of x, as soon as single tiles would be more workgroups than CUs (bf16
//    64 x 4096 x 4096: 15.5 and 19.6, 48 x 2048 x 2048: 5.3 and 6.6; with fewer, 16 x 2048 x 2048: 5.0 and 4.4), and 8 waves of
//    two slices, whose registers have room for it (64 x 8192 x 8192: bf16 40 and 47 with 16 waves, float32 83 and 106).
constexpr size_t STAGE_MOST = 64 << 10;
constexpr int CUS = 256;

template <typename E, int NT, int GATES, bool STAGED>
void launch(const Q4Dev& q, const Q4Call& a, int split, int waves, int most, size_t staged, hipStream_t s) {
    constexpr int gates = GATES ? GATES : 1;
    const dim3 grid(GATES ? q.tiles : (q.gates * q.tiles + NT - 1) / NT, (a.B + most - 1) / most), block(64 * waves * gates);
    const size_t lds = (size_t)split * gates * NT * 1024 * (STAGED ? 1 : Q4Type<E>::PARTS) + staged;
    if (q.per_block == 1) hipLaunchKernelGGL((wnv_q4_rows<E, NT, 1, GATES, STAGED>), grid, block, lds, s, q, a, split, waves, most);
    else if (q.per_block == 2) hipLaunchKernelGGL((wnv_q4_rows<E, NT, 2, GATES, STAGED>), grid, block, lds, s, q, a, split, waves, most);
    else hipLaunchKernelGGL((wnv_q4_rows<E, NT, 4, GATES, STAGED>), grid, block, lds, s, q, a, split, waves, most);
}
template <typename E, int GATES> void launch(const Q4Dev& q, const Q4Call& a, hipStream_t s) {
    constexpr int PARTS = Q4Type<E>::PARTS;
    const int slices = GATES == 0 ? 16 : GATES == 2 ? 8 : 4;    // a workgroup is 16 waves at most, 12 with three gates
    const int split = std::min(slices, q.kb), most = 16 / PARTS;
    const size_t staged = (size_t)PARTS * std::min(a.B, most) * (16 * q.kb + 1) * 16;
    const int64_t passes = (a.B + most - 1) / most;
    const bool pays = PARTS == 3 ? GATES || q.gates * q.tiles * passes <= 2 * CUS : a.B <= 16 && q.kb > split;
    if (staged <= STAGE_MOST && pays) return launch<E, 1, GATES, true>(q, a, split, split, most, staged, s);
    if constexpr (!GATES) {
        if ((int64_t)q.gates * q.tiles * ((a.B + 15) / 16) > CUS) return launch<E, 2, GATES, false>(q, a, split, std::min(split, 8), 16, 0, s);
    }
    launch<E, 1, GATES, false>(q, a, split, split, 16, 0, s);
}
template <typename E> void launch(const Q4Dev& q, const Q4Call& a, hipStream_t s) {
    if (!a.state) launch<E, 0>(q, a, s);
    else if (q.gates == 2) launch<E, 2>(q, a, s);
    else launch<E, 3>(q, a, s);
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
    q.tiles = (q.rows + 15) / 16; q.kb = (cin + 127) / 128; q.per_block = 128 / group;
    *out = h;
    return WNV_OK;
}

static wnv_status q4_pack(wnv_q4* h, const uint8_t* codes, const wnv_bf16* scales, const uint8_t* zeros, const float* bias, int* bad,
                          hipStream_t s) {
    Q4Dev& q = h->q;
    const size_t tiles = (size_t)q.gates * q.tiles, words = tiles * q.kb * 256, gs = tiles * q.kb * q.per_block * 16;
    HIP_TRY(hipDeviceSynchronize());    // steps under way on other streams still read what is about to be written over
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
    if (found) return fail(WNV_ERR_INVALID_ARG, "wnv_q4: a code or zero point is over 15, or a weight is not finite or over 3e38");
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
    WNV_BY_TYPE(dtype, launch<E>(h->q, a, (hipStream_t)stream));
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
    WNV_BY_TYPE(dtype, launch<E>(h->q, a, (hipStream_t)stream));
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
