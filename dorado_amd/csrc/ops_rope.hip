// dorado_amd/csrc/ops_rope.hip — mibc_rope: rotary positions of queries and keys in one launch.
//   (a, b) -> A (a cos t - b sin t, a sin t + b cos t),  t = position * frequency
// Bound by HBM: every element is read and written once.  What could bound it instead is the angle: at position 10^6 an f32
// product is off by 0.03 radians, so the angle is formed in f64 as TURNS (position * (frequency / 2 pi)), its whole turns are
// dropped exactly, and sine and cosine of the rest come from Taylor polynomials on an eighth of a turn to each side of the
// nearest quarter (error below 2e-9 and 2e-10).  A thread does that once for the 8 pairs it owns and applies it to every head
// of its token that it visits, so the ~250 instructions of 8 angles are spread over several heads.
// Measured: 64 x 1024 tokens x 16 heads of 64 f16 53 us (5.1 TB/s), 100001 tokens x 40 heads of 128 bf16, half of each rotated, 397 us
// (5.2 TB/s); a copy of that size runs at 4.6 - 5.4 TB/s.
#include "ops.h"

#include <math.h>
#include <string.h>

struct RopeArgs {
    mibc_rope_args a;
    int64_t total;      // batch * tokens
    int items;          // 16-column items of a head that are visited (rotated ones first)
    int rot_items;      // rot_dim / 16
    int threads;        // threads per token (a power of two, <= 256)
    int head_lanes;     // threads / items
};

__device__ __forceinline__ void rope_angle(double turns, float amplitude, float &c, float &s) {
    const float r = (float)(turns - rint(turns));            // [-1/2, 1/2]
    const float q = rintf(4.0f * r);                         // nearest quarter, -2 .. 2
    const float x = fmaf(q, -0.25f, r) * 6.283185307179586f; // [-pi/4, pi/4]; the fma is exact
    const float z = x * x;
    float sn = fmaf(z, 2.7557319e-6f, -1.9841270e-4f);       // 1/9!, 1/7!
    sn = fmaf(z, sn, 8.3333333e-3f);
    sn = fmaf(z, sn, -1.6666667e-1f);
    sn = fmaf(z * x, sn, x);
    float cs = fmaf(z, -2.7557319e-7f, 2.4801587e-5f);       // 1/10!, 1/8!
    cs = fmaf(z, cs, -1.3888889e-3f);
    cs = fmaf(z, cs, 4.1666667e-2f);
    cs = fmaf(z, cs, -0.5f);
    cs = fmaf(z, cs, 1.0f);
    const int k = (int)q & 3;
    const float c0 = (k & 1) ? sn : cs, s0 = (k & 1) ? cs : sn;
    c = ((k == 1 || k == 2) ? -c0 : c0) * amplitude;
    s = ((k & 2) ? -s0 : s0) * amplitude;
}
__device__ __forceinline__ double rope_position(const mibc_rope_args &a, int64_t at, int64_t t) {
    if (a.positions == nullptr) return (double)(a.start + t);
    return a.positions_64 ? (double)((const int64_t *)a.positions)[at] : (double)((const int32_t *)a.positions)[at];
}
#define ROPE_TURN 0.15915494309189535   // 1 / (2 pi)

// 16-byte accesses: a thread owns the 8 pairs of one item (half layout: 8 columns of each half; interleaved: 16 neighbouring
// columns) of the heads head_lane, head_lane + head_lanes, ... of one token
template <typename T, bool INTERLEAVED>
__global__ __launch_bounds__(256) void rope_kernel(RopeArgs r) {
    const mibc_rope_args &a = r.a;
    const int sub = threadIdx.x & (r.threads - 1);
    const int item = sub % r.items, head0 = sub / r.items;
    if (head0 >= r.head_lanes) return;
    const bool rotate = item < r.rot_items;
    const int c0 = (!rotate || INTERLEAVED) ? item * 16 : item * 8;
    const int c1 = (!rotate || INTERLEAVED) ? c0 + 8 : c0 + a.rot_dim / 2;
    double f[8];
    if (rotate) {
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = a.freqs[item * 8 + i] * ROPE_TURN;
    }
    const int per = 256 / r.threads;     // tokens per workgroup
    for (int64_t at = (int64_t)blockIdx.x * per + threadIdx.x / r.threads; at < r.total; at += (int64_t)gridDim.x * per) {
        const int64_t n = (unsigned)at / (unsigned)a.tokens;
        const int64_t t = at - n * a.tokens;
        float c[8], s[8];
        if (rotate) {
            const double p = rope_position(a, at, t);
#pragma unroll
            for (int i = 0; i < 8; ++i) rope_angle(p * f[i], a.amplitude, c[i], s[i]);
        }
#pragma unroll
        for (int w = 0; w < 2; ++w) {
            if (a.x[w] == nullptr) continue;
            const T *x = (const T *)a.x[w] + n * a.x_stride[w][0] + t * a.x_stride[w][1];
            T *o = (T *)a.out[w] + n * a.out_stride[w][0] + t * a.out_stride[w][1];
            for (int h = head0; h < a.heads[w]; h += r.head_lanes) {
                const T *xh = x + h * a.x_stride[w][2];
                T *oh = o + h * a.out_stride[w][2];
                float u[8], v[8];
                op_load8(xh + c0, u);
                op_load8(xh + c1, v);
                if (rotate) {
                    float y[8], z[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const float p = INTERLEAVED ? (i < 4 ? u[2 * i] : v[2 * i - 8]) : u[i];
                        const float q = INTERLEAVED ? (i < 4 ? u[2 * i + 1] : v[2 * i - 7]) : v[i];
                        const float yy = fmaf(p, c[i], -(q * s[i])), zz = fmaf(p, s[i], q * c[i]);
                        if (INTERLEAVED) {
                            if (i < 4) {
                                y[2 * i] = yy;
                                y[2 * i + 1] = zz;
                            } else {
                                z[2 * i - 8] = yy;
                                z[2 * i - 7] = zz;
                            }
                        } else {
                            y[i] = yy;
                            z[i] = zz;
                        }
                    }
                    op_store8<T>(oh + c0, y);
                    op_store8<T>(oh + c1, z);
                } else {
                    op_store8<T>(oh + c0, u);
                    op_store8<T>(oh + c1, v);
                }
            }
        }
    }
}

// any even rot_dim, any alignment: one thread per pair or copied column of a token, for ANY_HEADS heads (blockIdx.y): one angle for
// eight heads, eight pairs of 2- or 4-byte loads in flight (8 x 4096 tokens x 16 heads of 40 bf16 3.2 TB/s; one thread per pair of every
// head 1.4)
constexpr int ANY_HEADS = 8;
template <typename T>
__global__ __launch_bounds__(256) void rope_any_kernel(RopeArgs r) {
    const mibc_rope_args &a = r.a;
    const int half = a.rot_dim / 2, per = half + a.head_dim - a.rot_dim, heads = a.heads[0] + a.heads[1];
    const int64_t all = r.total * per;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < all; i += (int64_t)gridDim.x * 256) {
        const int64_t at = i / per, n = (unsigned)at / (unsigned)a.tokens, t = at - n * a.tokens;
        const int e = (int)(i - at * per);
        const bool rotate = e < half;
        const int ca = !rotate ? e + half : a.interleaved ? 2 * e : e, cb = !rotate ? ca : a.interleaved ? 2 * e + 1 : e + half;
        float c = 1.0f, s = 0.0f;
        if (rotate) rope_angle(rope_position(a, at, t) * (a.freqs[e] * ROPE_TURN), a.amplitude, c, s);
        T p[ANY_HEADS], q[ANY_HEADS];
        auto place = [&](int i, bool out) {
            const int hh = min(blockIdx.y * ANY_HEADS + i, (unsigned)heads - 1), w = hh >= a.heads[0], h = w ? hh - a.heads[0] : hh;
            const int64_t *st = out ? a.out_stride[w] : a.x_stride[w];
            return (T *)(out ? a.out[w] : (void *)a.x[w]) + n * st[0] + t * st[1] + h * st[2];
        };
#pragma unroll
        for (int i = 0; i < ANY_HEADS; ++i) {
            const T *x = place(i, false);
            p[i] = x[ca];
            q[i] = x[cb];
        }
#pragma unroll
        for (int i = 0; i < ANY_HEADS; ++i) {
            if ((int)blockIdx.y * ANY_HEADS + i >= heads) break;
            T *o = place(i, true);
            const float u = (float)p[i], v = (float)q[i];
            o[ca] = rotate ? (T)fmaf(u, c, -(v * s)) : p[i];
            if (rotate) o[cb] = (T)fmaf(u, s, v * c);
        }
    }
}

static int rope_check(const mibc_rope_args &a, bool *vec) {
    if (a.type != MIBC_TYPE_F16 && a.type != MIBC_TYPE_BF16 && a.type != MIBC_TYPE_F32)
        return op_refuse(MIBC_NOT_SUPPORTED, "rope: type must be f16, bf16 or f32");
    if (a.batch < 0 || a.tokens < 0 || a.heads[0] < 1 || a.heads[1] < 0) return op_refuse(MIBC_ERR_ARG, "rope: negative size, or no heads");
    if (a.head_dim < 2 || a.rot_dim < 2 || a.rot_dim % 2 != 0 || a.rot_dim > a.head_dim)
        return op_refuse(MIBC_ERR_ARG, "rope: rot_dim must be even, at least 2 and at most head_dim");
    if (a.head_dim > 4096 || (int64_t)a.heads[0] + a.heads[1] > 65536) return op_refuse(MIBC_NOT_SUPPORTED, "rope: head_dim <= 4096, heads <= 65536");
    if ((a.x[1] == nullptr) != (a.heads[1] == 0)) return op_refuse(MIBC_ERR_ARG, "rope: heads[1] must be 0 exactly where x[1] is NULL");
    if (!(fabsf(a.amplitude) <= 3.4e38f)) return op_refuse(MIBC_ERR_ARG, "rope: amplitude must be finite");
    if (a.batch == 0 || a.tokens == 0) return MIBC_OK;
    if (a.batch > 0x7fffffff || a.tokens > 0x7fffffff || a.batch * a.tokens > 0x7fffffff)
        return op_refuse(MIBC_NOT_SUPPORTED, "rope: at most 2^31 - 1 tokens");
    if (a.freqs == nullptr || !op_aligned(a.freqs, 8)) return op_refuse(MIBC_ERR_ARG, "rope: freqs must be f64 [rot_dim / 2]");
    if (a.positions != nullptr && !op_aligned(a.positions, a.positions_64 ? 8 : 4)) return op_refuse(MIBC_ERR_ARG, "rope: positions not aligned");
    const unsigned eb = (unsigned)op_type_bytes(a.type);
    *vec = a.head_dim % 16 == 0 && a.rot_dim % 16 == 0 && a.head_dim <= 1024;
    for (int w = 0; w < 2; ++w) {
        if (a.heads[w] == 0) continue;
        if (a.x[w] == nullptr || a.out[w] == nullptr) return op_refuse(MIBC_ERR_ARG, "rope: null pointer");
        if (!op_aligned(a.x[w], eb) || !op_aligned(a.out[w], eb)) return op_refuse(MIBC_ERR_ARG, "rope: pointer not aligned to its type");
        const int64_t size[3] = {a.batch, a.tokens, a.heads[w]};
        for (int d = 0; d < 3; ++d) {
            if (a.x_stride[w][d] < 0) return op_refuse(MIBC_ERR_ARG, "rope: negative stride");
            if (size[d] > 1 && a.out_stride[w][d] < a.head_dim) return op_refuse(MIBC_ERR_ARG, "rope: output heads overlap");
            if ((size[d] > 1 && a.x_stride[w][d] % 8 != 0) || (size[d] > 1 && a.out_stride[w][d] % 8 != 0)) *vec = false;
        }
        if (!op_aligned(a.x[w], 16) || !op_aligned(a.out[w], 16)) *vec = false;
    }
    auto span = [&](const void *p, int w, const int64_t *s) {
        return op_span(p, (int64_t)a.head_dim * eb, a.batch, s[0] * eb, a.tokens, s[1] * eb, a.heads[w], s[2] * eb);
    };
    const OpSpan x[2] = {span(a.x[0], 0, a.x_stride[0]), span(a.x[1], 1, a.x_stride[1])};
    const OpSpan out[2] = {span(a.out[0], 0, a.out_stride[0]), span(a.heads[1] ? a.out[1] : nullptr, 1, a.out_stride[1])};
    const OpSpan p = op_span(a.positions, a.batch * a.tokens * (a.positions_64 ? 8 : 4)), f = op_span(a.freqs, (int64_t)a.rot_dim * 4);
    if (!op_plain(out[0]) || (a.heads[1] && !op_plain(out[1]))) return op_refuse(MIBC_ERR_ARG, "rope: output heads overlap");
    bool fine = op_apart(out[0], out[1]);
    for (int w = 0; w < 2; ++w)
        fine = fine && (op_same(out[w], x[w]) || op_apart(out[w], x[w])) && op_apart(out[w], x[1 - w]) && op_apart(out[w], p) && op_apart(out[w], f);
    if (!fine) return op_refuse(MIBC_ERR_ARG, "rope: an output may be its input, but not overlap it, another operand or the other output otherwise");
    return MIBC_OK;
}

template <typename T>
static hipError_t rope_launch(hipStream_t s, RopeArgs &r, bool vec) {
    const mibc_rope_args &a = r.a;
    const int heads = a.heads[0] + a.heads[1];
    if (!vec) {
        const int64_t all = r.total * (a.rot_dim / 2 + a.head_dim - a.rot_dim);
        const int64_t blocks = (all + 255) / 256;
        const dim3 grid((unsigned)(blocks < 65536 ? blocks : 65536), (unsigned)((heads + ANY_HEADS - 1) / ANY_HEADS));
        return op_launch(rope_any_kernel<T>, grid, 256, 0, s, r);
    }
    bool inplace = true;
    for (int w = 0; w < 2; ++w)
        if (a.heads[w]) inplace = inplace && a.x[w] == a.out[w] && memcmp(a.x_stride[w], a.out_stride[w], sizeof(a.x_stride[w])) == 0;
    r.rot_items = a.rot_dim / 16;
    r.items = inplace ? r.rot_items : a.head_dim / 16;
    // as few threads per token as give each at least one item of every fourth head: the angles of a thread serve several heads
    int threads = 1;
    while (threads < 256 && (threads < r.items || threads * 4 < r.items * heads)) threads *= 2;
    r.threads = threads;
    r.head_lanes = threads / r.items;
    const int per = 256 / threads;
    const int64_t blocks = (r.total + per - 1) / per;
    const int64_t most = (int64_t)mibc_ncu() * 32;   // a workgroup walks several tokens: frequencies are read once
    const dim3 grid((unsigned)(blocks < most ? blocks : most));
    return a.interleaved ? op_launch(rope_kernel<T, true>, grid, 256, 0, s, r) : op_launch(rope_kernel<T, false>, grid, 256, 0, s, r);
}

static int rope_run(hipStream_t s, const mibc_rope_args &a, bool vec) {
    RopeArgs r{};
    r.a = a;
    r.total = a.batch * a.tokens;
#define ROPE_T(T) rope_launch<T>(s, r, vec)
    return op_hip(a.type == MIBC_TYPE_F16 ? ROPE_T(half_t) : a.type == MIBC_TYPE_BF16 ? ROPE_T(bf16_t) : ROPE_T(float), "rope");
#undef ROPE_T
}

// launch on a stream of the current device (the engine's own path); checks included
int mibc_launch_rope(hipStream_t s, const mibc_rope_args &a) {
    bool vec = false;
    if (const int rc = rope_check(a, &vec)) return rc;
    return a.batch == 0 || a.tokens == 0 ? MIBC_OK : rope_run(s, a, vec);
}

extern "C" int mibc_rope(int device, void *stream, const mibc_rope_args *a) {
    if (a == nullptr) return op_refuse(MIBC_ERR_ARG, "rope: null arguments");
    bool vec = false;
    if (const int rc = rope_check(*a, &vec)) return rc;
    if (a->batch == 0 || a->tokens == 0) return MIBC_OK;
    OpDevice d(device);
    if (d.rc != hipSuccess) return op_hip(d.rc, "rope: device");
    return rope_run((hipStream_t)stream, *a, vec);
}

extern "C" int mibc_rope_frequencies(int scaling, int rot_dim, double theta, double factor, double original_length, double turns_low,
                                     double turns_high, double *freqs) {
    if (rot_dim < 2 || rot_dim % 2 != 0 || freqs == nullptr) return op_refuse(MIBC_ERR_ARG, "rope_frequencies: rot_dim must be even");
    if (!(theta > 0.0) || !(theta < 1e300)) return op_refuse(MIBC_ERR_ARG, "rope_frequencies: theta must be positive");
    if (scaling < MIBC_ROPE_PLAIN || scaling > MIBC_ROPE_BY_PARTS) return op_refuse(MIBC_NOT_SUPPORTED, "rope_frequencies: unknown scaling");
    if (scaling != MIBC_ROPE_PLAIN && (!(factor > 0.0) || !(factor < 1e300)))
        return op_refuse(MIBC_ERR_ARG, "rope_frequencies: factor must be positive");
    if (scaling == MIBC_ROPE_BASE && rot_dim == 2) return op_refuse(MIBC_ERR_ARG, "rope_frequencies: a larger base needs rot_dim > 2");
    if (scaling == MIBC_ROPE_BY_PARTS && (!(original_length > 0.0) || !(turns_high > turns_low)))
        return op_refuse(MIBC_ERR_ARG, "rope_frequencies: original_length > 0 and turns_high > turns_low");
    const double base = scaling == MIBC_ROPE_BASE ? theta * pow(factor, (double)rot_dim / (rot_dim - 2)) : theta;
    for (int i = 0; i < rot_dim / 2; ++i) {
        double f = pow(base, -2.0 * i / rot_dim);
        if (scaling == MIBC_ROPE_LINEAR) f /= factor;
        if (scaling == MIBC_ROPE_BY_PARTS) {
            double keep = (original_length * f * ROPE_TURN - turns_low) / (turns_high - turns_low);
            keep = keep < 0.0 ? 0.0 : keep > 1.0 ? 1.0 : keep;
            f *= keep + (1.0 - keep) / factor;
        }
        freqs[i] = f;
    }
    return MIBC_OK;
}
