// dorado_amd/csrc/ops_norm.hip — mibc_rms_norm: residual addition, RMS norm and an optional 8-bit output in one pass.
//   h = x + alpha r,   y = h / sqrt(sum h^2 / C + eps) * w,   q = rne(y / s), s = max|y| / 127 | 448
// A few flops per element against 2-8 bytes: bound by HBM.  So a row is read once, stays in f32 registers (TPR threads hold
// NCH chunks of 8 consecutive columns each) through both reductions (sum of squares, then max |y| where the output has 8 bits)
// and leaves once.  Rows of up to 2048 columns take one wave, or as few of its lanes as hold them (2M rows of 32 bf16: 4 lanes 6.5 TB/s,
// 16 lanes 2.6), and reduce by lane shuffles alone; wider ones
// take a workgroup and one LDS exchange per reduction: as few threads as hold the row in six chunks (11320 columns: 256 threads x 6
// chunks 39 us, 1024 x 2 54), 1024 beyond.
// Measured: 262144 x 512 f16 with residual 134 us (6.0 TB/s), 16383 x 4096 bf16 with residual, sum and e4m3 codes per 128 columns
// 90 us (5.3 TB/s), 10000 x 5001 bf16 with residual (unaligned rows) 73 us (4.1 TB/s), 3794 x 11320 e4m3 38 us (3.4 TB/s: the
// conversion's instructions, of which the quotients' last step is 1 us).
#include "ops.h"

struct NormArgs {
    mibc_rms_norm_args a;
};

template <typename T, bool VEC>
__device__ __forceinline__ void norm_load(const T *row, int col, int cols, float v[8]) {
    if (VEC) {
        op_load8(row + col, v);
    } else if (col + 8 <= cols) {
        op_load8<true>(row + col, v);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = (col + i < cols) ? (float)row[col + i] : 0.0f;
    }
}
template <typename T, bool VEC>
__device__ __forceinline__ void norm_store(T *row, int col, int cols, const float v[8]) {
    if (VEC) {
        op_store8<T>(row + col, v);
    } else if (col + 8 <= cols) {
        op_store8<T, true>(row + col, v);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (col + i < cols) row[col + i] = (T)v[i];
    }
}

// over the TPR threads that hold a row; `red`: one slot per wave
template <int TPR>
__device__ __forceinline__ float norm_reduce_sum(float v, float *red) {
#pragma unroll
    for (int o = (TPR < 64 ? TPR : 64) / 2; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    if (TPR > 64) {
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
        __syncthreads();
        v = red[0];
#pragma unroll
        for (int i = 1; i < TPR / 64; ++i) v += red[i];
    }
    return v;
}
template <int TPR>
__device__ __forceinline__ unsigned norm_reduce_max(unsigned v, unsigned *red) {
#pragma unroll
    for (int o = (TPR < 64 ? TPR : 64) / 2; o > 0; o >>= 1) v = max(v, (unsigned)__shfl_xor((int)v, o, 64));
    if (TPR > 64) {
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
        __syncthreads();
        v = red[0];
#pragma unroll
        for (int i = 1; i < TPR / 64; ++i) v = max(v, red[i]);
    }
    return v;
}

template <typename T, int TPR, int NCH, bool VEC>
__global__ __launch_bounds__(TPR > 256 ? TPR : 256) void rms_norm_kernel(NormArgs n) {
    constexpr int NT = TPR > 256 ? TPR : 256;
    __shared__ float red[2][NT / 64];
    const mibc_rms_norm_args &a = n.a;
    const int lane = threadIdx.x % TPR;
    const int64_t row = (((int64_t)blockIdx.y << 20) + blockIdx.x) * (NT / TPR) + threadIdx.x / TPR;
    if (row >= a.rows) return;     // whole rows of lanes, or a whole workgroup
    const int cols = a.cols;
    const T *x = (const T *)a.x + row * a.x_stride;
    const T *r = (const T *)a.residual + row * a.residual_stride;
    float h[NCH][8];
    float ss = 0.0f;
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
        const int col = (lane + i * TPR) * 8;
#pragma unroll
        for (int e = 0; e < 8; ++e) h[i][e] = 0.0f;
        if (col < cols) norm_load<T, VEC>(x, col, cols, h[i]);
    }
    if (a.residual != nullptr) {
#pragma unroll
        for (int i = 0; i < NCH; ++i) {
            const int col = (lane + i * TPR) * 8;
            if (col < cols) {
                float v[8];
                norm_load<T, VEC>(r, col, cols, v);
#pragma unroll
                for (int e = 0; e < 8; ++e) h[i][e] = fmaf(a.alpha, v[e], h[i][e]);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < NCH; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e) ss = fmaf(h[i][e], h[i][e], ss);
    if (a.sum_out != nullptr) {
        T *o = (T *)a.sum_out + row * a.sum_stride;
#pragma unroll
        for (int i = 0; i < NCH; ++i) {
            const int col = (lane + i * TPR) * 8;
            if (col < cols) norm_store<T, VEC>(o, col, cols, h[i]);
        }
    }
    ss = norm_reduce_sum<TPR>(ss, red[0]);
    const float rstd = 1.0f / sqrtf(ss / (float)cols + a.eps);
    // y replaces h
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
        const int col = (lane + i * TPR) * 8;
        float w[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) w[e] = 1.0f;
        if (a.weight != nullptr && col < cols) {
            if (a.weight_type == MIBC_TYPE_F32)
                norm_load<float, VEC>((const float *)a.weight, col, cols, w);
            else
                norm_load<T, VEC>((const T *)a.weight, col, cols, w);
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) h[i][e] = h[i][e] * rstd * w[e];
    }
    if (a.out_type == a.type) {
        T *o = (T *)a.out + row * a.out_stride;
#pragma unroll
        for (int i = 0; i < NCH; ++i) {
            const int col = (lane + i * TPR) * 8;
            if (col < cols) norm_store<T, VEC>(o, col, cols, h[i]);
        }
        return;
    }
    // 8-bit output.  Magnitudes are compared as whole numbers: NaN and infinity are larger than every finite value then
    unsigned top[NCH];
    unsigned all = 0;
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
        top[i] = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) top[i] = max(top[i], __float_as_uint(h[i][e]) & 0x7fffffffu);   // columns behind the row hold zeros
        all = max(all, top[i]);
    }
    const float most = a.out_type == MIBC_TYPE_I8 ? 127.0f : 448.0f;
    if (a.group == 0) {
        all = norm_reduce_max<TPR>(all, (unsigned *)red[1]);
#pragma unroll
        for (int i = 0; i < NCH; ++i) top[i] = all;
    } else {   // a group is group / 8 = 4, 8 or 16 neighbouring lanes of one chunk index
#pragma unroll
        for (int i = 0; i < NCH; ++i)
#pragma unroll
            for (int o = 1; o < 16; o <<= 1) {
                const unsigned w = (unsigned)__shfl_xor((int)top[i], o, 64);
                top[i] = (o * 8 < a.group) ? max(top[i], w) : top[i];
            }
    }
    uint8_t *o = (uint8_t *)a.out + row * a.out_stride;
    float *sc = a.scale_out + row * a.scale_stride;
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
        const int chunk = lane + i * TPR, col = chunk * 8;
        if (col >= cols) continue;
        const bool fine = top[i] < 0x7f800000u;
        float s = fine ? __uint_as_float(top[i]) / most : NAN;
        if (s == 0.0f) s = 1.0f;     // nothing but zeros, or values whose scale is below f32
        unsigned lo = 0, hi = 0;
        if (fine) {
            // y / s, rounded once: the product with the rounded reciprocal is off by a step or two, its remainder is exact, and one
            // more product with the reciprocal sets it right
            float v[8];              // at most 127 or 448 times 1 + 2^-23: rounds to the largest code
            const auto divide = [&](float by) {
                const float inv = 1.0f / by;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float q = h[i][e] * inv;
                    v[e] = fmaf(fmaf(-q, by, h[i][e]), inv, q);
                }
            };
            if (s >= 1e-20f) {
                divide(s);
            } else {                 // remainders and reciprocals beyond f32: both sides are lifted by 2^64 first
#pragma unroll
                for (int e = 0; e < 8; ++e) h[i][e] *= 0x1p64f;
                divide(s * 0x1p64f);
                // a scale of few bits is off by up to a third
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = fminf(fmaxf(v[e], -most), most);
            }
            if (a.out_type == MIBC_TYPE_I8) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    lo |= ((unsigned)(int)rintf(v[e]) & 0xffu) << (8 * e);
                    hi |= ((unsigned)(int)rintf(v[4 + e]) & 0xffu) << (8 * e);
                }
            } else {                 // the conversion's NaN range begins above 464
                lo = __builtin_amdgcn_cvt_pk_fp8_f32(v[0], v[1], lo, false);
                lo = __builtin_amdgcn_cvt_pk_fp8_f32(v[2], v[3], lo, true);
                hi = __builtin_amdgcn_cvt_pk_fp8_f32(v[4], v[5], hi, false);
                hi = __builtin_amdgcn_cvt_pk_fp8_f32(v[6], v[7], hi, true);
            }
        }
        if (VEC) {
            *(uintx2 *)(o + col) = (uintx2){lo, hi};
        } else if (col + 8 <= cols) {
            op_put<uintx2, true>(o + col, (uintx2){lo, hi});
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (col + e < cols) o[col + e] = (uint8_t)((e < 4 ? lo : hi) >> (8 * (e & 3)));
        }
        if (a.group == 0 ? chunk == 0 : col % a.group == 0) sc[a.group == 0 ? 0 : col / a.group] = s;
    }
}

template <typename T, bool VEC>
static hipError_t norm_launch(hipStream_t s, const NormArgs &n) {
    const int chunks = (n.a.cols + 7) / 8;
    const int64_t rows = n.a.rows;
    // a launch holds less than 2^32 threads in x
#define NORM_GO(TPR, NCH, NT)                                                                                        \
    do {                                                                                                             \
        const int64_t blocks = (rows + NT / TPR - 1) / (NT / TPR), x = blocks < 1 << 20 ? blocks : 1 << 20;          \
        return op_launch(rms_norm_kernel<T, TPR, NCH, VEC>, dim3((unsigned)x, (unsigned)((blocks + x - 1) / x)), NT, 0, s, n); \
    } while (0)
    if (chunks <= 4) NORM_GO(4, 1, 256);
    if (chunks <= 8) NORM_GO(8, 1, 256);
    if (chunks <= 16) NORM_GO(16, 1, 256);
    if (chunks <= 64) NORM_GO(64, 1, 256);
    if (chunks <= 128) NORM_GO(64, 2, 256);
    if (chunks <= 256) NORM_GO(64, 4, 256);
    if (chunks <= 512) NORM_GO(256, 2, 256);
    if (chunks <= 1024) NORM_GO(256, 4, 256);
    if (chunks <= 1536) NORM_GO(256, 6, 256);
    NORM_GO(1024, 4, 1024);
#undef NORM_GO
}

static int norm_check(const mibc_rms_norm_args &a, bool *vec) {
    if (a.type != MIBC_TYPE_F16 && a.type != MIBC_TYPE_BF16 && a.type != MIBC_TYPE_F32)
        return op_refuse(MIBC_NOT_SUPPORTED, "rms_norm: type must be f16, bf16 or f32");
    if (a.rows < 0 || a.cols < 1) return op_refuse(MIBC_ERR_ARG, "rms_norm: rows >= 0 and cols >= 1");
    if (a.cols > 32768) return op_refuse(MIBC_NOT_SUPPORTED, "rms_norm: at most 32768 columns");
    if (a.rows > (int64_t)0x7fffffff) return op_refuse(MIBC_NOT_SUPPORTED, "rms_norm: at most 2^31 - 1 rows");
    if (a.weight != nullptr && a.weight_type != MIBC_TYPE_F32 && a.weight_type != a.type)
        return op_refuse(MIBC_NOT_SUPPORTED, "rms_norm: weight must be f32 or of the input's type");
    const bool quant = a.out_type == MIBC_TYPE_I8 || a.out_type == MIBC_TYPE_E4M3;
    if (!quant && a.out_type != a.type) return op_refuse(MIBC_NOT_SUPPORTED, "rms_norm: output is of the input's type, int8 or e4m3");
    if (quant) {
        if (a.group != 0 && a.group != 32 && a.group != 64 && a.group != 128)
            return op_refuse(MIBC_NOT_SUPPORTED, "rms_norm: group must be 0 (a row), 32, 64 or 128");
        if (a.group != 0 && a.cols % a.group != 0) return op_refuse(MIBC_ERR_ARG, "rms_norm: cols must be a multiple of group");
    } else if (a.group != 0) {
        return op_refuse(MIBC_ERR_ARG, "rms_norm: group needs an 8-bit output");
    }
    if (!(a.eps >= 0.0f)) return op_refuse(MIBC_ERR_ARG, "rms_norm: eps must not be negative");
    if (a.reserved != 0) return op_refuse(MIBC_ERR_ARG, "rms_norm: reserved must be 0");
    if (a.rows == 0) return MIBC_OK;
    if (a.x == nullptr || a.out == nullptr || (quant && a.scale_out == nullptr))
        return op_refuse(MIBC_ERR_ARG, "rms_norm: null pointer");
    const int ngroups = a.group == 0 ? 1 : a.cols / a.group;
    if (a.rows > 1 && (a.out_stride < a.cols || (a.sum_out != nullptr && a.sum_stride < a.cols) || (quant && a.scale_stride < ngroups)))
        return op_refuse(MIBC_ERR_ARG, "rms_norm: output rows overlap");
    if (a.x_stride < 0 || a.residual_stride < 0) return op_refuse(MIBC_ERR_ARG, "rms_norm: negative stride");
    const unsigned eb = (unsigned)op_type_bytes(a.type);
    if (!op_aligned(a.x, eb) || !op_aligned(a.residual, eb) || !op_aligned(a.sum_out, eb) || !op_aligned(a.weight, (unsigned)op_type_bytes(a.weight_type)) ||
        !op_aligned(a.out, (unsigned)op_type_bytes(a.out_type)) || !op_aligned(a.scale_out, 4))
        return op_refuse(MIBC_ERR_ARG, "rms_norm: pointer not aligned to its type");
    const int64_t wide = (int64_t)a.cols * eb, ob = op_type_bytes(a.out_type);
    const OpSpan x = op_span(a.x, wide, a.rows, a.x_stride * eb), r = op_span(a.residual, wide, a.rows, a.residual_stride * eb),
                 w = op_span(a.weight, (int64_t)a.cols * op_type_bytes(a.weight_type)), sum = op_span(a.sum_out, wide, a.rows, a.sum_stride * eb),
                 out = op_span(a.out, a.cols * ob, a.rows, a.out_stride * ob), sc = op_span(a.scale_out, ngroups * 4, quant ? a.rows : 0, a.scale_stride * 4);
    auto in_place = [&](const OpSpan &o) { return (op_same(o, x) || op_apart(o, x)) && (op_same(o, r) || op_apart(o, r)) && op_apart(o, w); };
    if (!in_place(sum) || !in_place(out) || !op_apart(sum, out) || !op_apart(sc, x) || !op_apart(sc, r) || !op_apart(sc, w) || !op_apart(sc, sum) ||
        !op_apart(sc, out))
        return op_refuse(MIBC_ERR_ARG, "rms_norm: an output may be x or residual, but not overlap them, the weight or another output otherwise");
    // aligned 16-byte accesses where every row of every tensor allows them, unaligned ones and single elements at a row's end elsewhere
    *vec = a.cols % 8 == 0 && op_aligned(a.x, 16) && a.x_stride % 8 == 0 && op_aligned(a.weight, 16) &&
           (a.residual == nullptr || (op_aligned(a.residual, 16) && a.residual_stride % 8 == 0)) &&
           (a.sum_out == nullptr || (op_aligned(a.sum_out, 16) && a.sum_stride % 8 == 0)) &&
           op_aligned(a.out, quant ? 8 : 16) && a.out_stride % 8 == 0;
    return MIBC_OK;
}

static int norm_run(hipStream_t s, const mibc_rms_norm_args &a, bool vec) {
    const NormArgs n{a};
#define NORM_T(T) (vec ? norm_launch<T, true>(s, n) : norm_launch<T, false>(s, n))
    return op_hip(a.type == MIBC_TYPE_F16 ? NORM_T(half_t) : a.type == MIBC_TYPE_BF16 ? NORM_T(bf16_t) : NORM_T(float), "rms_norm");
#undef NORM_T
}

// launch on a stream of the current device (the engine's own path); checks included
int mibc_launch_rms_norm(hipStream_t s, const mibc_rms_norm_args &a) {
    bool vec = false;
    if (const int rc = norm_check(a, &vec)) return rc;
    return a.rows == 0 ? MIBC_OK : norm_run(s, a, vec);
}

extern "C" int mibc_rms_norm(int device, void *stream, const mibc_rms_norm_args *a) {
    if (a == nullptr) return op_refuse(MIBC_ERR_ARG, "rms_norm: null arguments");
    bool vec = false;
    if (const int rc = norm_check(*a, &vec)) return rc;
    if (a->rows == 0) return MIBC_OK;
    OpDevice d(device);
    if (d.rc != hipSuccess) return op_hip(d.rc, "rms_norm: device");
    return norm_run((hipStream_t)stream, *a, vec);
}
