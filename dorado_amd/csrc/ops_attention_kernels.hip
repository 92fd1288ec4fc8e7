// dorado_amd/csrc/ops_attention_kernels.hip — the kernels of mibc_attention for one head size (ATT_D, set by the Makefile).
#include "ops_attention.h"

#ifndef ATT_D
#error "compile with -DATT_D=<head size>"
#endif

typedef bf16_t bf16x8_t __attribute__((ext_vector_type(8)));
typedef short short4_att __attribute__((ext_vector_type(4)));
#define LDSP(T) __attribute__((address_space(3))) T *
typedef __attribute__((address_space(3))) void *att_lds_vptr;
typedef const __attribute__((address_space(1))) char *att_gptr;

// The matrix instructions take weights in the type of v: 2^LIFT times exp(score - the running maximum), which is only moved when it grew
// by more than 2^GROW, so that most tiles rescale nothing.  f16 ends at 2^16 and drops what is below 2^-25: with 2^11 and 2^4 a weight is
// off by at most 2^-36 of the largest (2^17 such keys by 2^-19), whereas 2^0 and 2^8 lost 0.2 % of the mass of 131072 keys 18 below a
// single one.  2^13 and 2^2 rescale more often (4 x 16 heads x 4096 of 64 with scores of spread 4: 345 us against 342).  bf16 has f32's range,
// so sums of its values may end beyond f32: where one did, the pass for values that are not finite runs at 2^-40 (2^28 keys of weight 2^8
// stay below 2^-4 of the largest value; values below 2^-86 lose bits beside such sums).
// The exponent is one fma of the raw score and minus the maximum, which was rounded: all weights of a row are off by one factor, which
// cancels, but whose own exponent is up to 2^-25 of the maximum.  Rows whose maximum is at FAR or beyond, where it nears what the type
// holds, take the other pass too; a score is rounded like the maximum there before the two are subtracted.
template <typename T>
struct AttType;
template <>
struct AttType<half_t> {
    typedef half8_t vec8;
    static constexpr unsigned EXPONENT = 0x7c00, MANTISSA = 0x03ff, ONE = 0x3c00;
    static constexpr float LIFT = 11.0f, LIFT_AGAIN = 11.0f, GROW = 4.0f, FAR = 0x1p22f;
    static __device__ __forceinline__ float16_t mfma32(vec8 a, vec8 b, float16_t c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
    static __device__ __forceinline__ float4_t mfma16(vec8 a, vec8 b, float4_t c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
};
template <>
struct AttType<bf16_t> {
    typedef bf16x8_t vec8;
    static constexpr unsigned EXPONENT = 0x7f80, MANTISSA = 0x007f, ONE = 0x3f80;
    static constexpr float LIFT = 0.0f, LIFT_AGAIN = -40.0f, GROW = 8.0f, FAR = 0x1p28f;
    static __device__ __forceinline__ float16_t mfma32(vec8 a, vec8 b, float16_t c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
    static __device__ __forceinline__ float4_t mfma16(vec8 a, vec8 b, float4_t c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
};

// 16 bytes per lane from base + offset straight to LDS at `lds_addr` + 16 * lane (one wait state between M0 and its use).  Written
// as assembly, because the compiler waits for every LDS load of its own before any LDS read, and the next tile's are meant to
// stay in flight: the kernels wait for them by vmcnt.  The load writes no register.  M0 is one the compiler never allocates (it takes no
// clobber of it either) and needs for nothing else here: a test looks at the assembly for that.
__device__ __forceinline__ void att_dma16(att_gptr base, unsigned offset, unsigned lds_addr) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds_addr), "v"(offset), "s"(base) : "memory");
}
template <typename V8>
__device__ __forceinline__ V8 att_lds16(unsigned addr) {
    return *(LDSP(const V8))(size_t)addr;
}
// 4 rows x 16 columns per 16 lanes: lane l hands in the address of row l / 4, columns 4 (l & 3) .. + 3, and gets column l of the 4 rows
__device__ __forceinline__ uintx2 att_lds_tr(unsigned addr) {
    return __builtin_bit_cast(uintx2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((LDSP(short4_att))(size_t)addr));
}
#define ATT_FENCE() __builtin_amdgcn_sched_barrier(0)     // the compiler moves nothing across

__device__ __forceinline__ float att_exp2(float x) { return __builtin_amdgcn_exp2f(x); }
// f x for weights f >= 0: an infinity that a row sees stays one, also where the weight is 0 in f32
__device__ __forceinline__ float att_weigh(float f, float x) { return __builtin_isinf(x) ? x : f * x; }
// over the two half waves
__device__ __forceinline__ float att_half_max(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float att_half_add(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ int att_low_half(int x) {   // lane i and i + 32 get lane i's
    return (int)__builtin_amdgcn_permlane32_swap((unsigned)x, (unsigned)x, false, false)[0];
}

// What a row sees: [lo, hi) and, if `apart` kernels ask for it, [plo, phi), the prefix.  Both borders of both grow with the token
// (documents in order), so the rows between two rows see nothing outside [lo of the first, hi of the last) and the prefixes' hull.
struct AttRow {
    int lo, hi, plo, phi, pos;
};
// borders <= t, t the same in all lanes: 64 borders a step
__device__ __forceinline__ int att_borders(const int32_t *border, int count, int t, int lane) {
    int base = 0;
    while (count > 64) {
        const int stride = (count + 63) >> 6;       // lane's block of borders: is its last one <= t?
        const int k = __popcll(__ballot(border[base + min((lane + 1) * stride, count) - 1] <= t));
        const int skip = min(k * stride, count);
        base += skip;
        count = min(stride, count - skip);
    }
    const bool in = lane < count && border[base + min(lane, max(count - 1, 0))] <= t;
    return base + __popcll(__ballot(in));
}
// where in the borders a token's document lies: its index, start and end (no document: an empty one)
struct AttDoc {
    int index, start, end;
};
__device__ __forceinline__ AttDoc att_doc(const mibc_attention_args &a, int t, int borders, int at, int next) {
    AttDoc d;     // borders out of order end in some document, whose keys are clamped all the same
    d.index = min(max(borders - 1, 0), a.n_docs);
    d.start = min(max(at, 0), a.k_tokens);
    d.end = borders > 0 && d.index < a.n_docs ? min(max(next, d.start), a.k_tokens) : d.start;
    return d;
}
__device__ __forceinline__ AttRow att_row(const AttArgs &p, int b, int t, const AttDoc &doc) {
    const mibc_attention_args &a = p.a;
    int k0 = 0, k1, pre = 0;
    AttRow r;
    if (a.doc_offsets != nullptr) {
        k0 = doc.start;
        k1 = doc.end;
        if (a.prefix != nullptr && k1 > k0) pre = a.prefix[doc.index];
        r.pos = t;
    } else {
        k1 = a.k_len != nullptr ? min(max(a.k_len[b], 0), a.k_tokens) : a.k_tokens;
        r.pos = (a.q_start == MIBC_ATTN_END ? k1 - a.q_tokens : a.q_start) + t;
        if (a.prefix != nullptr) pre = a.prefix[b];
    }
    const int lo = p.back < 0 ? k0 : min(max(k0, r.pos - p.back), k1);
    const int hi = p.ahead < 0 ? k1 : max(min(k1, r.pos + p.ahead + 1), k0);
    const int ph = k0 + min(max(pre, 0), k1 - k0);
    const bool join = ph >= lo;          // the prefix reaches the window
    r.lo = join ? k0 : lo;
    r.hi = join ? max(hi, ph) : hi;
    r.plo = k0;
    r.phi = ph;
    return r;
}

// The kernel's arguments, read again where they are next needed: kept in scalar registers over the main loop they spill
__device__ __forceinline__ const AttArgs &att_args_again() {
    auto at = __builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(at));
    return *(const AttArgs *)at;
}

// workgroups i and i + 8 of 16 go to one XCD: they get neighbouring pairs
__device__ __forceinline__ int att_twin(const AttArgs &p, unsigned x) { return p.twin ? (x & ~15u) | (x & 7) << 1 | (x >> 3 & 1) : x; }

// The exponent (base 2) of a score is mul * x + add, x being what the registers hold.  A slope adds slope * |i - j| to x, in x's unit.
//   no cap:   x = q.k, mul = scale log2(e)
//   ATT_NEAR: cap tanh(y) = cap - 2 cap / (1 + e^2y), so x = 1 / (1 + e^2y) and the last product is the exponent's own fma; the
//             largest score is the smallest x.  Two numbers of the cap's size cancel: off by up to cap 2^-21 whatever the score, so
//             this form is for caps up to 64 (in tiles of rows, where the other one costs half as much again)
//   ATT_FAR:  x = q.k tanh(y) / y, mul = scale log2(e): off by 2^-20 of the score.  Below |y| = 1/2 the Taylor series of
//             tanh(y) / y up to y^12 (the next term is below 2^-23), above it cap / scale (1 - e^-2|y|) / (1 + e^-2|y|)
template <int CAP, bool SLOPES>
struct AttScore {
    float mul, add, slope, in, most;
    static constexpr float HIDDEN = CAP == ATT_NEAR ? INFINITY : -INFINITY;
    __device__ __forceinline__ AttScore(const AttArgs &p, int head) {
        mul = CAP == ATT_NEAR ? -2.0f * p.cap_out : p.scale2;
        add = CAP == ATT_NEAR ? p.cap_out : 0.0f;
        in = p.cap_in;
        most = p.cap_out;
        slope = SLOPES ? -p.a.slopes[head] * 1.4426950408889634f / mul : 0.0f;
    }
    __device__ __forceinline__ float capped(float x) const {
        if (CAP == ATT_NEAR) return __builtin_amdgcn_rcpf(1.0f + att_exp2(x * in));
        const float y = x * in, z = y * y;
        float t = fmaf(z, 3.592128036572481e-3f, -8.863235529902197e-3f);      // 21844 / 6081075, -1382 / 155925
        t = fmaf(z, t, 2.186948853615520e-2f);                                 // 62 / 2835
        t = fmaf(z, t, -5.396825396825397e-2f);                                // -17 / 315
        t = fmaf(z, t, 0.1333333333333333f);
        t = fmaf(z, t, -0.3333333333333333f);
        t = fmaf(z, t, 1.0f);
        const float e = att_exp2(fabsf(y) * -2.8853900817779268f);             // 2 log2(e)
        const float far = copysignf(most * (1.0f - e) * __builtin_amdgcn_rcpf(1.0f + e), x);
        return fabsf(y) < 0.5f ? x * t : far;                                  // NaN: far, which is NaN
    }
    // of the raw score x; off: minus the maximum, in the first pass with what else is added to the exponent
    template <bool SAFE>
    __device__ __forceinline__ float weight(float x, float off, float lift) const {
        return SAFE ? att_exp2((fmaf(x, mul, add) + off) + lift) : att_exp2(fmaf(x, mul, off));
    }
    __device__ __forceinline__ float larger(float a, float b) const { return CAP == ATT_NEAR ? fminf(a, b) : fmaxf(a, b); }
};

template <typename T>
__device__ __forceinline__ bool att_far(float m) {     // a row's maximum, which may be -infinity (no key) or not a number
    return fabsf(m) >= AttType<T>::FAR && !__builtin_isinf(m);
}
// 1 where a value is NaN (kind 0), infinity (1), -infinity (2), else 0
template <typename T>
__device__ __forceinline__ uintx4 att_places(uintx4 v, int kind) {
    typedef AttType<T> X;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        unsigned w = 0;
#pragma unroll
        for (int z = 0; z < 2; ++z) {
            const unsigned x = v[e] >> (16 * z);
            const bool odd = (x & X::EXPONENT) == X::EXPONENT;
            const int is = (x & X::MANTISSA) ? 0 : (x & 0x8000u) ? 2 : 1;
            w |= odd && is == kind ? X::ONE << (16 * z) : 0u;
        }
        v[e] = w;
    }
    return v;
}

// ------------------------------------------------------------------------------------------------------------------
// Row tiles of 128 rows: four waves of 32, all over the same tiles of 64 keys in LDS (two stages, filled by direct
// global -> LDS loads while the tile before is worked on).
//   S^T[key][row] = K Q^T   on 32x32x16: lane (row = lane & 31, half = lane >> 5) holds keys 8 g + 4 half + 0..3 of each 32
//   O^T[dim][row] = V^T P^T  takes P^T from those very registers: the 16 k-slots of a step are enumerated as the keys a lane holds,
//   and V^T comes out of the row-major V tile through transposing LDS reads (ds_read_b64_tr_b16).
// P is rounded to the type of v for that product, which takes one type for both operands; the sums l are of the unrounded values.  Two
// parts of P would be exact to f32 for half as many matrix instructions again, which is what bounds this kernel: the rounding makes the
// result's error against 64 bits 1.2 - 1.4 times that of the output's own rounding (f16 2.1e-4 -> 2.5 - 2.9e-4, bf16 1.5e-3 -> 1.9e-3).
// A row's maximum and sum are one lane pair's: no exchange but one half-wave swap per tile.  Operands are read four instructions
// ahead, and the products of 16 keys with V run beside the probabilities of the next 16.
// Head size 128: the matrix pipe works 0.54 of the cycles beside 170 plain instructions per tile and wave (1024 matrix cycles), and power
// holds the clock at 1.7 GHz: 8192 x 16 heads 496 - 515 us, causal 16384 x 16 heads 996 - 1030 us (1060 - 1104 TFLOP/s over two cards; a
// library product of 8192^3 1229).  Capped scores, 298 plain instructions (an exponential and a reciprocal more per score): causal
// 1157 - 1212 us (906 - 950 TFLOP/s).  Head size 64, as many exponentials for half the products: 4 x 16 heads x 4096 321 us
// (856 TFLOP/s), with three waves per SIMD; two 334 us.
template <int D>
__device__ __forceinline__ int att_k_slot(int row, int chunk) {   // 16-byte column of the K tile in LDS
    return D == 128 ? chunk ^ (row & 15) : D == 64 ? chunk ^ ((row >> 1) & 7) : chunk ^ ((row >> 2) & 3);
}
template <int D>
__device__ __forceinline__ int att_v_slot(int row, int chunk) {
    return D == 128 ? chunk ^ ((row & 3) << 2) : D == 64 ? chunk ^ (((row >> 1) & 1) << 2) : chunk;
}

template <typename T, int D, int CAP, bool SLOPES>
__global__ __launch_bounds__(256, D <= 64 ? 3 : 2) void attention_kernel(AttArgs p) {
    typedef AttType<T> X;
    typedef typename X::vec8 vec8;
    constexpr int NT = 256, ROWS = 128;
    constexpr int PITCH = D * 2;
    constexpr int TILE = 64 * PITCH;
    constexpr int CH = TILE / 16;               // 16-byte pieces of a tile
    constexpr int NLD = (CH + NT - 1) / NT;
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    __shared__ int flag;                        // some wave's result is not finite
    const unsigned lds = (unsigned)(size_t)(LDSP(unsigned char))smem;
    const mibc_attention_args &a = p.a;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int half = lane >> 5;

    // workgroup -> (split, tile, pair)
    const unsigned id = (blockIdx.y << 20) + blockIdx.x;
    if (id >= p.groups) return;
    int pair, tile, split;
    if (p.order == 0) {
        const unsigned rest = p.by_pairs.div(id);
        pair = att_twin(p, id - rest * p.pairs);
        const unsigned z = p.by_splits.div(rest);
        split = rest - z * p.splits;
        tile = p.tiles - 1 - (int)z;                    // causal: the long tiles start first
    } else {
        const unsigned rest = id >> (p.twin ? 4 : 3), y = p.by_splits.div(rest), z = p.by_tiles.div(y);
        split = rest - y * p.splits;
        tile = y - z * p.tiles;
        pair = p.twin ? att_twin(p, z * 16 + (id & 15)) : z * 8 + (id & 7);
    }
    const int b = p.by_kv.div(pair), kvh = pair - b * a.kv_heads;

    // lanes 32 and 33 look at the workgroup's first and last row instead of their own
    const int row = tile * ROWS + wave * 32 + (lane & 31);
    const int rr = min(row, p.rows - 1), t = p.by_group.div(rr), head = kvh * p.group + (rr - t * p.group);
    const int t_first = p.by_group.div(tile * ROWS), t_last = p.by_group.div(min(tile * ROWS + ROWS, p.rows) - 1);
    const int tt = lane == 32 ? t_first : lane == 33 ? t_last : t;
    AttDoc doc{};
    if (a.doc_offsets != nullptr) {
        const int n = a.n_docs + 1, w_first = __builtin_amdgcn_readfirstlane(t), w_last = __builtin_amdgcn_readlane(t, 31);
        int borders, f, g, at, next;
        if (n <= 64) {      // all borders in the lanes: one load
            const int mine = a.doc_offsets[min(lane, n - 1)];
            auto upto = [&](int x) { return (int)__popcll(__ballot(lane < n && mine <= x)); };
            const int first = upto(w_first), last = upto(w_last);
            borders = first;
            for (int i = first; i < last; ++i) borders += __builtin_amdgcn_readlane(mine, i) <= t;     // borders between the wave's rows
            f = upto(t_first);
            g = upto(t_last);
            borders = lane == 32 ? f : lane == 33 ? g : borders;
            const int d = min(max(borders - 1, 0), n - 1);
            at = __shfl(mine, d, 64);
            next = __shfl(mine, min(d + 1, n - 1), 64);
        } else {
            borders = att_borders(a.doc_offsets, n, w_first, lane);
            for (int i = borders; i < n; ++i) {
                const int x = a.doc_offsets[i];
                if (x > w_last) break;
                if (x <= t) ++borders;
            }
            f = att_borders(a.doc_offsets, n, t_first, lane);
            g = att_borders(a.doc_offsets, n, t_last, lane);
            borders = lane == 32 ? f : lane == 33 ? g : borders;
            const int d = min(max(borders - 1, 0), n - 1);
            at = a.doc_offsets[d];
            next = a.doc_offsets[min(d + 1, n - 1)];
        }
        doc = att_doc(a, tt, borders, at, next);
    }
    AttRow see = att_row(p, b, tt, doc);
    int w0 = __builtin_amdgcn_readlane(see.lo, 32), w1 = __builtin_amdgcn_readlane(see.hi, 33);
    int p0 = __builtin_amdgcn_readlane(see.plo, 32), p1 = __builtin_amdgcn_readlane(see.phi, 33);
    const bool apart = a.prefix != nullptr && p.back >= 0;
    // tiles of the prefix, then of the window; one range where their tiles would overlap
    int np = apart && p0 < p1 ? (p1 - p0 + 63) >> 6 : 0;
    if (np > 0 && p0 + 64 * np > w0) {
        w0 = min(w0, p0);
        w1 = max(w1, p1);
        np = 0;
    }
    const int ntiles = np + (w0 < w1 ? (w1 - w0 + 63) >> 6 : 0);
    int it0 = 0, it1 = ntiles;
    if (p.splits > 1) {
        it0 = (int)p.by_splits.div((unsigned)ntiles * split);      // ntiles * splits < 2^31
        it1 = (int)p.by_splits.div((unsigned)ntiles * (split + 1));
    }
    // the wave's rows: outside [lo_min, hi_max) no row sees a key, inside [lo_max, hi_min) every row sees it
    see.lo = att_low_half(see.lo);
    see.hi = att_low_half(see.hi);
    see.plo = att_low_half(see.plo);
    see.phi = att_low_half(see.phi);
    see.pos = att_low_half(see.pos);
    const int lo_min = __builtin_amdgcn_readfirstlane(see.lo), lo_max = __builtin_amdgcn_readlane(see.lo, 31);
    const int hi_min = __builtin_amdgcn_readfirstlane(see.hi), hi_max = __builtin_amdgcn_readlane(see.hi, 31);
    const int plo_min = __builtin_amdgcn_readfirstlane(see.plo), phi_max = apart ? __builtin_amdgcn_readlane(see.phi, 31) : 0;

    // pieces of a tile this thread moves: LDS order is linear in the thread, the swizzle permutes what is fetched.  Where the
    // rows that all threads move at once are whole periods of the swizzle, the pieces of a thread differ by the row alone
    constexpr bool EVEN = NT % (D / 8) == 0 && NT / (D / 8) % 16 == 0;
    const att_gptr kb = (att_gptr)a.k + (b * a.k_stride[0] + kvh * a.k_stride[2]) * 2;
    const att_gptr vb = (att_gptr)a.v + (b * a.v_stride[0] + kvh * a.v_stride[2]) * 2;
    const unsigned krow = (unsigned)a.k_stride[1] * 2, vrow = (unsigned)a.v_stride[1] * 2;
    unsigned koff[EVEN ? 1 : NLD], voff[EVEN ? 1 : NLD];
#pragma unroll
    for (int i = 0; i < (EVEN ? 1 : NLD); ++i) {
        const int c = i * NT + tid, r = c / (D / 8), s = c % (D / 8);
        koff[i] = r * krow + att_k_slot<D>(r, s) * 16;
        voff[i] = r * vrow + att_v_slot<D>(r, s) * 16;
    }
    auto first_key = [&](int it) { return it < np ? p0 + 64 * it : w0 + 64 * (it - np); };
    auto fetch = [&](int it, int stage) {
        const int j0 = first_key(it), left = (it < np ? p1 : w1) - j0;
        const att_gptr kt = kb + (int64_t)j0 * krow, vt = vb + (int64_t)j0 * vrow;
        const unsigned to = lds + stage * (2 * TILE) + wave * 1024;
#pragma unroll
        for (int i = 0; i < NLD; ++i)
            if (i * NT + wave * 64 < CH) {
                const unsigned at = to + i * (NT * 16);
                if (left >= 64) {
                    const int more = EVEN ? i * (NT / (D / 8)) : 0;
                    att_dma16(kt + (int64_t)more * krow, koff[EVEN ? 0 : i], at);
                    att_dma16(vt + (int64_t)more * vrow, voff[EVEN ? 0 : i], at + TILE);
                } else {   // rows behind the last key repeat it: nobody sees them
                    const int c = i * NT + tid, r = c / (D / 8), s = c % (D / 8), rc = min(r, left - 1);
                    att_dma16(kt, rc * krow + att_k_slot<D>(r, s) * 16, at);
                    att_dma16(vt, rc * vrow + att_v_slot<D>(r, s) * 16, at + TILE);
                }
            }
    };

    if (it0 < it1) fetch(it0, 0);
    if (tid == 0) flag = 0;
    vec8 qf[D / 16];
    {
        const T *q = (const T *)a.q + b * a.q_stride[0] + t * a.q_stride[1] + head * a.q_stride[2] + 8 * half;
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) qf[ks] = *(const vec8 *)(q + 16 * ks);
    }
    // fragment addresses of this lane in stage 0
    unsigned kaddr[D / 16], vaddr[D / 32];
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks) kaddr[ks] = lds + (lane & 31) * PITCH + att_k_slot<D>(lane & 31, 2 * ks + half) * 16;
#pragma unroll
    for (int db = 0; db < D / 32; ++db) {
        const int r = 4 * half + ((lane >> 2) & 3);
        vaddr[db] = lds + TILE + r * PITCH + att_v_slot<D>(r, 4 * db + 2 * ((lane >> 4) & 1) + ((lane >> 1) & 1)) * 16 + (lane & 1) * 8;
    }
    const AttScore<CAP, SLOPES> score(p, head);

    float16_t o[D / 32], s[2];
    float m, l;
    auto start = [&]() {
#pragma unroll
        for (int db = 0; db < D / 32; ++db) o[db] = (float16_t)(0.0f);
        m = -INFINITY;
        l = 0.0f;
    };
    // operands are read four instructions ahead of their use (the fences keep the compiler from moving reads down to it)
    auto products = [&](unsigned at) {
        constexpr int N = D / 8;
        auto key = [&](int i) { return att_lds16<vec8>(kaddr[i >> 1] + (at + (i & 1) * (32 * PITCH))); };
        vec8 kf[4];
        s[0] = s[1] = (float16_t)(0.0f);
#pragma unroll
        for (int i = 0; i < 4; ++i) kf[i] = key(i);
        ATT_FENCE();
#pragma unroll
        for (int i = 0; i < N; ++i) {
            s[i & 1] = X::mfma32(kf[i & 3], qf[i >> 1], s[i & 1]);
            if (i + 4 < N) kf[i & 3] = key(i + 4);
            if (i & 1) ATT_FENCE();
        }
    };
    // element e = 32 i + (r & 3) + 8 (r >> 2) of a tile is key j0 + 4 half + e
#define ATT_EACH                             \
    _Pragma("unroll") for (int i = 0; i < 2; ++i) \
    _Pragma("unroll") for (int r = 0, e = 32 * i; r < 16; ++r, e = 32 * i + (r & 3) + 8 * (r >> 2))
    auto shape = [&](int j0) {      // raw products -> what AttScore calls x
        if (CAP) {
            ATT_EACH s[i][r] = score.capped(s[i][r]);
        }
        if (SLOPES) {
            const float away = (float)(see.pos - j0 - 4 * half);
            ATT_EACH s[i][r] = fmaf(score.slope, fabsf(away - (float)e), s[i][r]);
        }
    };
    // what a row does not see leaves its scores; returns the bits 16 i + r of what it sees
    auto hide_all = [&](int j0) {
        const int at0 = j0 + 4 * half, lo = see.lo - at0, hi = see.hi - at0, plo = apart ? see.plo - at0 : 0, phi = apart ? see.phi - at0 : 0;
        unsigned seen = 0;
        ATT_EACH {
            const bool v = ((e >= lo) & (e < hi)) | ((e >= plo) & (e < phi));
            s[i][r] = v ? s[i][r] : score.HIDDEN;
            seen |= v ? 1u << (16 * i + r) : 0u;
        }
        return seen;
    };
    auto hide = [&](int j0) {
        const int at0 = j0 + 4 * half, lo = see.lo - at0, hi = see.hi - at0;
        if (apart) {
            (void)hide_all(j0);
        } else {
            if (j0 + 64 > hi_min) {
                ATT_EACH s[i][r] = e < hi ? s[i][r] : score.HIDDEN;
            }
            if (j0 < lo_max) {
                ATT_EACH s[i][r] = e >= lo ? s[i][r] : score.HIDDEN;
            }
        }
    };
    float off;
    auto maxima = [&](auto safe_) {     // safe_: o may hold infinities
        float top = s[0][0];
        ATT_EACH top = score.larger(top, s[i][r]);
        top = att_half_max(fmaf(top, score.mul, score.add));
        if (__any(top > m + X::GROW)) {
            const float mn = fmaxf(m, top);
            const float f = m == -INFINITY ? 0.0f : att_exp2(m - mn);
            m = mn;
            l *= f;
#pragma unroll
            for (int db = 0; db < D / 32; ++db)
#pragma unroll
                for (int r = 0; r < 16; ++r) o[db][r] = decltype(safe_)::value ? att_weigh(f, o[db][r]) : o[db][r] * f;
        }
        off = (decltype(safe_)::value ? 0.0f : score.add + X::LIFT) - (m == -INFINITY ? 0.0f : m);
    };
    auto probabilities = [&](auto safe_, int k) {       // of 16 keys
        constexpr bool SAFE = decltype(safe_)::value;
        uintx4 w;
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float x = score.template weight<SAFE>(s[k >> 1][8 * (k & 1) + 2 * i], off, X::LIFT_AGAIN);
            const float y = score.template weight<SAFE>(s[k >> 1][8 * (k & 1) + 2 * i + 1], off, X::LIFT_AGAIN);
            sum += x + y;                   // before the rounding: the sum is also a result
            w[i] = op_pack2(x, y, T());
        }
        l += sum;
        return __builtin_bit_cast(vec8, w);
    };
    auto values = [&](unsigned at, int db, int k) {      // V^T operand: 32 dims x 16 keys
        const uintx2 x = att_lds_tr(vaddr[db] + (at + k * (16 * PITCH))), y = att_lds_tr(vaddr[db] + (at + k * (16 * PITCH) + 8 * PITCH));
        return (uintx4){x[0], x[1], y[0], y[1]};
    };
    auto step = [&](auto stage_, int it) {
        constexpr unsigned AT = decltype(stage_)::value * (2 * TILE);
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        const int j0 = first_key(it);
        if ((j0 >= hi_max || j0 + 64 <= lo_min) && (j0 >= phi_max || j0 + 64 <= plo_min)) {      // no row of the wave
            if (it + 1 < it1) fetch(it + 1, decltype(stage_)::value ^ 1);
            return;
        }
        products(AT);
        if (it + 1 < it1) fetch(it + 1, decltype(stage_)::value ^ 1);      // behind the reads of K, which it would hold up
        shape(j0);
        if (j0 < lo_max || j0 + 64 > hi_min) hide(j0);
        maxima(std::false_type());
        // the products of 16 keys run beside the probabilities of the next 16, whose values are read meanwhile
        // two waves per SIMD (head sizes from 96): the one that forms probabilities goes first; both pipes have work from it then,
        // and the other's score products fill the matrix pipe meanwhile (causal 16384 x 16 heads of 128: 1053 -> 1030 us, capped
        // 1267 -> 1211).  With three, windows and documents lose 3 % by it
        if (D > 64) __builtin_amdgcn_s_setprio(1);
        constexpr int N = D / 32;
        uintx4 v[2][N];
#pragma unroll
        for (int db = 0; db < N; ++db) v[0][db] = values(AT, db, 0);
        vec8 pf[2];
        pf[0] = probabilities(std::false_type(), 0);
        ATT_FENCE();
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if (k < 3) {
#pragma unroll
                for (int db = 0; db < N; ++db) v[(k + 1) & 1][db] = values(AT, db, k + 1);
                pf[(k + 1) & 1] = probabilities(std::false_type(), k + 1);
            }
#pragma unroll
            for (int db = 0; db < N; ++db) o[db] = X::mfma32(__builtin_bit_cast(vec8, v[k & 1][db]), pf[k & 1], o[db]);
            ATT_FENCE();
            if (D > 64 && k == 2) __builtin_amdgcn_s_setprio(0);
        }
    };
    start();
    for (int it = it0; it < it1; it += 2) {
        step(std::integral_constant<int, 0>(), it);
        if (it + 1 < it1) step(std::integral_constant<int, 1>(), it + 1);
    }
    float zero[4] = {0.0f, 0.0f, 0.0f, 0.0f};      // 0 * x: 0, or NaN where x is not finite
#pragma unroll
    for (int db = 0; db < D / 32; ++db)
#pragma unroll
        for (int r = 0; r < 16; ++r) zero[r & 3] = fmaf(o[db][r], 0.0f, zero[r & 3]);
    const bool odd = !(zero[0] + zero[1] + zero[2] + zero[3] == 0.0f) || att_far<T>(m);
    if (__any(odd) && lane == 0) flag = 1;
    __syncthreads();
    if (flag) {
        // something is not finite: from a value or key that the row sees, 0 * (a value that it does not see), or a sum beyond f32; or a
        // maximum is too far out.  Once more, tile by tile: values that are not finite stay out of the products, and the places of NaN (kind 0), infinity (1) and
        // -infinity (2) are multiplied with the mask instead, so that they reach the rows that see their key and no other
        start();
#pragma unroll 1
        for (int it = it0; it < it1; ++it) {
            __syncthreads();
            fetch(it, 0);
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            __syncthreads();
            const int j0 = first_key(it);
            products(0);
            shape(j0);
            const unsigned seen = hide_all(j0);
            maxima(std::true_type());
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const vec8 pf = probabilities(std::true_type(), k);
                uintx4 w;
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    w[e] = ((seen >> (8 * k + 2 * e)) & 1 ? X::ONE : 0u) | ((seen >> (8 * k + 2 * e + 1)) & 1 ? X::ONE << 16 : 0u);
                const vec8 vis = __builtin_bit_cast(vec8, w);
#pragma unroll
                for (int db = 0; db < D / 32; ++db) {
                    const uintx4 v = values(0, db, k);
                    uintx4 fine = v;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        if ((v[e] & X::EXPONENT) == X::EXPONENT) fine[e] &= 0xffff0000u;
                        if (((v[e] >> 16) & X::EXPONENT) == X::EXPONENT) fine[e] &= 0x0000ffffu;
                    }
                    o[db] = X::mfma32(__builtin_bit_cast(vec8, fine), pf, o[db]);
#pragma unroll 1
                    for (int kind = 0; kind < 3; ++kind) {
                        const float what = kind == 0 ? NAN : kind == 1 ? INFINITY : -INFINITY;
                        const float16_t hit = X::mfma32(__builtin_bit_cast(vec8, att_places<T>(v, kind)), vis, (float16_t)(0.0f));
#pragma unroll
                        for (int r = 0; r < 16; ++r)
                            if (hit[r] > 0.0f) o[db][r] += what;
                    }
                }
            }
        }
    }

    l = att_half_add(l);
    const float base = m == -INFINITY ? 0.0f : m;
    const float inv = l == 0.0f ? 0.0f : __builtin_amdgcn_rcpf(l);
    l *= att_exp2(flag ? -X::LIFT_AGAIN : -X::LIFT);
    {   // row, token and head are worked out again rather than kept in registers over the loop
        const AttArgs &p = att_args_again();
        const mibc_attention_args &a = p.a;
        const int row = tile * ROWS + wave * 32 + (lane & 31);
        if (row >= p.rows) return;
        const int t = p.by_group.div(row), head = kvh * p.group + (row - t * p.group);
        if (p.splits > 1) {
            const int64_t at = ((int64_t)pair * p.rows + row) * p.splits + split;
            float *po = p.part_o + at * D + 4 * half;
#pragma unroll
            for (int db = 0; db < D / 32; ++db)
#pragma unroll
                for (int g = 0; g < 4; ++g)
                    *(floatx4 *)(po + 32 * db + 8 * g) = (floatx4){o[db][4 * g] * inv, o[db][4 * g + 1] * inv, o[db][4 * g + 2] * inv, o[db][4 * g + 3] * inv};
            if (half == 0) p.part_l[at] = l == 0.0f ? -INFINITY : base + log2f(l);
            return;
        }
        T *out = (T *)a.out + b * a.out_stride[0] + t * a.out_stride[1] + head * a.out_stride[2] + 4 * half;
#pragma unroll
        for (int db = 0; db < D / 32; ++db)
#pragma unroll
            for (int g = 0; g < 4; ++g)
                *(uintx2 *)(out + 32 * db + 8 * g) = (uintx2){op_pack2(o[db][4 * g] * inv, o[db][4 * g + 1] * inv, T()),
                                                              op_pack2(o[db][4 * g + 2] * inv, o[db][4 * g + 3] * inv, T())};
        if (a.lse != nullptr && half == 0)
            a.lse[((int64_t)b * a.heads + head) * a.q_tokens + t] = l == 0.0f ? -INFINITY : base * 0.6931471805599453f + logf(l);
    }
}

// ------------------------------------------------------------------------------------------------------------------
// At most 16 rows per (batch, key head) pair: single tokens and short runs of them over long caches.  Bound by reading K and V
// once, so nothing is shared between waves and nothing waits for a barrier: each of the four waves walks its own steps of 32 keys
// (wave w the steps w, w + 4, ...), K straight into matrix operands, V through two private LDS stages (transposing reads).  The
// next step's loads leave as soon as the scores have used up the K operands: 16 KB of a wave are in flight all the time but for
// the few hundred cycles of its score instructions, 128 KB per CU.  16x16x32 instructions: S^T[key][row], lane (row = lane & 15,
// quarter = lane >> 4) holds keys 4 quarter + 0..3 of each 16, which are its k-slots in O^T[dim][row] = V^T P^T.  Matrix work is
// free here, so P goes in as two 16-bit parts (value and remainder): the result is rounded once, at the end.
// Measured: 48 x 8 pairs over 2048 .. 8192 keys of 128 bf16 219 us (5.0 TB/s), one token of 2 pairs over 131072 keys 32 us, 32 x 16 pairs
// over 4096 keys of 64 f16 109 us (4.9 TB/s).
template <int D>
__device__ __forceinline__ int att_v_slot16(int row, int chunk) {
    return D == 128 ? chunk ^ (((row & 3) << 2) | ((row & 4) >> 1)) : D == 64 ? chunk ^ ((((row >> 1) & 1) << 2) | ((row & 4) >> 1)) : chunk;
}

template <typename T, int D, int CAP, bool SLOPES>
__global__ __launch_bounds__(256, 2) void attention_token_kernel(AttArgs p) {
    typedef AttType<T> X;
    typedef typename X::vec8 vec8;
    constexpr int PITCH = D * 2;
    constexpr int STAGE = 32 * PITCH;
    constexpr int NV = STAGE / 1024;            // LDS loads of a step
    constexpr int NK = D / 32;                  // K operand pieces of 16 keys
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    const unsigned lds = (unsigned)(size_t)(LDSP(unsigned char))smem;
    const mibc_attention_args &a = p.a;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int l15 = lane & 15, quarter = lane >> 4;
    const unsigned id = (blockIdx.y << 20) + blockIdx.x;
    if (id >= p.groups) return;
    const int split = p.by_pairs.div(id), pair = att_twin(p, id - split * p.pairs);
    const int b = p.by_kv.div(pair), kvh = pair - b * a.kv_heads;

    const int rr = min(l15, p.rows - 1), t = p.by_group.div(rr), head = kvh * p.group + (rr - t * p.group);
    AttDoc doc{};
    if (a.doc_offsets != nullptr) {
        int borders = 0;
        for (int i = 0; i < a.n_docs + 1 && a.doc_offsets[i] < a.q_tokens; ++i) borders += a.doc_offsets[i] <= t;   // at most 16 tokens
        const int d = min(max(borders - 1, 0), a.n_docs);
        doc = att_doc(a, t, borders, a.doc_offsets[d], a.doc_offsets[min(d + 1, a.n_docs)]);
    }
    const AttRow see = att_row(p, b, t, doc);
    // rows grow with the lane up to the last, which lane 15 repeats
    const int lo_min = __builtin_amdgcn_readfirstlane(see.lo), lo_max = __builtin_amdgcn_readlane(see.lo, 15);
    const int hi_min = __builtin_amdgcn_readfirstlane(see.hi), hi_max = __builtin_amdgcn_readlane(see.hi, 15);
    const int p0 = __builtin_amdgcn_readfirstlane(see.plo), p1 = __builtin_amdgcn_readlane(see.phi, 15);
    const bool apart = a.prefix != nullptr && p.back >= 0;
    int w0 = lo_min, w1 = hi_max, np = apart && p0 < p1 ? (p1 - p0 + 31) >> 5 : 0;
    if (np > 0 && p0 + 32 * np > w0) {
        w0 = min(w0, p0);
        w1 = max(w1, p1);
        np = 0;
    }
    const int steps = np + (w0 < w1 ? (w1 - w0 + 31) >> 5 : 0);
    const int it0 = (int)p.by_splits.div((unsigned)steps * split) + wave;      // steps * splits < 2^31
    const int it1 = (int)p.by_splits.div((unsigned)steps * (split + 1));

    vec8 qf[NK];
    {
        const T *q = (const T *)a.q + b * a.q_stride[0] + t * a.q_stride[1] + head * a.q_stride[2] + 8 * quarter;
#pragma unroll
        for (int kb = 0; kb < NK; ++kb) qf[kb] = *(const vec8 *)(q + 32 * kb);
    }
    const att_gptr kb0 = (att_gptr)a.k + (b * a.k_stride[0] + kvh * a.k_stride[2]) * 2;
    const att_gptr vb0 = (att_gptr)a.v + (b * a.v_stride[0] + kvh * a.v_stride[2]) * 2;
    const unsigned krow = (unsigned)a.k_stride[1] * 2, vrow = (unsigned)a.v_stride[1] * 2;
    const unsigned mine = lds + wave * (2 * STAGE);
    auto first_key = [&](int it) { return it < np ? p0 + 32 * it : w0 + 32 * (it - np); };
    auto fetch = [&](int it, vec8 (&kf)[2][NK], int stage) {
        const int j0 = first_key(it), last = min(32, (it < np ? p1 : w1) - j0) - 1;    // rows behind the last key repeat it
        const att_gptr kt = kb0 + (int64_t)j0 * krow, vt = vb0 + (int64_t)j0 * vrow;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const unsigned at = min(16 * i + l15, last) * krow + 16 * quarter;
#pragma unroll
            for (int kb = 0; kb < NK; ++kb) kf[i][kb] = *(const __attribute__((address_space(1))) vec8 *)(kt + (at + 64 * kb));
        }
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = i * 64 + lane, r = c / (D / 8), s = c % (D / 8);
            att_dma16(vt, min(r, last) * vrow + att_v_slot16<D>(r, s) * 16, mine + stage * STAGE + i * 1024);
        }
    };
    unsigned vaddr[D / 16];
#pragma unroll
    for (int db = 0; db < D / 16; ++db) {
        const int r = 4 * quarter + (l15 >> 2);
        vaddr[db] = mine + r * PITCH + att_v_slot16<D>(r, 2 * db + ((lane >> 1) & 1)) * 16 + (lane & 1) * 8;
    }
    const AttScore<CAP, SLOPES> score(p, head);

    float4_t o[D / 16];
    float m, l;
    auto pass = [&](auto safe_) {
        constexpr bool SAFE = decltype(safe_)::value;
#pragma unroll
        for (int db = 0; db < D / 16; ++db) o[db] = (float4_t)(0.0f);
        m = -INFINITY;
        l = 0.0f;
        vec8 kf[2][NK];
        if (it0 < it1) fetch(it0, kf, 0);
        for (int it = it0; it < it1; it += 4) {
            const int stage = ((it - it0) >> 2) & 1;
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            const int j0 = first_key(it);
            float4_t s[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                s[i] = (float4_t)(0.0f);
#pragma unroll
                for (int kb = 0; kb < NK; ++kb) s[i] = X::mfma16(kf[i][kb], qf[kb], s[i]);
            }
            if (it + 4 < it1) fetch(it + 4, kf, stage ^ 1);
            if (CAP) {
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int r = 0; r < 4; ++r) s[i][r] = score.capped(s[i][r]);
            }
            if (SLOPES) {
                const float away = (float)(see.pos - j0 - 4 * quarter);
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int r = 0; r < 4; ++r) s[i][r] = fmaf(score.slope, fabsf(away - (float)(16 * i + r)), s[i][r]);
            }
            unsigned seen = 0xff;
            if (SAFE || j0 < lo_max || j0 + 32 > hi_min) {
                seen = 0;
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const int j = j0 + 16 * i + 4 * quarter + r;
                        const bool v = (unsigned)(j - see.lo) < (unsigned)(see.hi - see.lo) || (unsigned)(j - see.plo) < (unsigned)(see.phi - see.plo);
                        s[i][r] = v ? s[i][r] : score.HIDDEN;
                        seen |= v ? 1u << (4 * i + r) : 0u;
                    }
            }
            float top = s[0][0];
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int r = 0; r < 4; ++r) top = score.larger(top, s[i][r]);
            top = fmaf(top, score.mul, score.add);
            if (__any(top > m + X::GROW)) {     // m is the row's, the same in its four lanes
                top = fmaxf(top, __shfl_xor(top, 16, 64));
                top = fmaxf(top, __shfl_xor(top, 32, 64));
                const float mn = fmaxf(m, top);
                const float f = m == -INFINITY ? 0.0f : att_exp2(m - mn);
                m = mn;
                l *= f;
#pragma unroll
                for (int db = 0; db < D / 16; ++db)
#pragma unroll
                    for (int r = 0; r < 4; ++r) o[db][r] = SAFE ? att_weigh(f, o[db][r]) : o[db][r] * f;
            }
            const float off = (SAFE ? 0.0f : score.add + X::LIFT) - (m == -INFINITY ? 0.0f : m);
            uintx4 hi, lo;
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int r = 0; r < 4; r += 2) {
                    const float x = score.template weight<SAFE>(s[i][r], off, X::LIFT_AGAIN), y = score.template weight<SAFE>(s[i][r + 1], off, X::LIFT_AGAIN);
                    l += x + y;
                    const unsigned h = op_pack2(x, y, T());
                    hi[2 * i + (r >> 1)] = h;
                    const T *hx = (const T *)&h;
                    lo[2 * i + (r >> 1)] = op_pack2(x - (float)hx[0], y - (float)hx[1], T());
                }
#pragma unroll
            for (int db = 0; db < D / 16; ++db) {
                const uintx2 x = att_lds_tr(vaddr[db] + stage * STAGE), y = att_lds_tr(vaddr[db] + stage * STAGE + 16 * PITCH);
                uintx4 v = {x[0], x[1], y[0], y[1]};
                if (SAFE) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        if ((v[e] & X::EXPONENT) == X::EXPONENT) v[e] &= 0xffff0000u;
                        if (((v[e] >> 16) & X::EXPONENT) == X::EXPONENT) v[e] &= 0x0000ffffu;
                    }
                }
                o[db] = X::mfma16(__builtin_bit_cast(vec8, v), __builtin_bit_cast(vec8, hi), o[db]);
                o[db] = X::mfma16(__builtin_bit_cast(vec8, v), __builtin_bit_cast(vec8, lo), o[db]);
            }
            if (SAFE) {   // as in attention_kernel
                uintx4 w;
#pragma unroll
                for (int e = 0; e < 4; ++e) w[e] = ((seen >> (2 * e)) & 1 ? X::ONE : 0u) | ((seen >> (2 * e + 1)) & 1 ? X::ONE << 16 : 0u);
#pragma unroll 1
                for (int kind = 0; kind < 3; ++kind)
#pragma unroll
                    for (int db = 0; db < D / 16; ++db) {
                        const uintx2 x = att_lds_tr(vaddr[db] + stage * STAGE), y = att_lds_tr(vaddr[db] + stage * STAGE + 16 * PITCH);
                        const uintx4 v = {x[0], x[1], y[0], y[1]};
                        const float4_t hit = X::mfma16(__builtin_bit_cast(vec8, att_places<T>(v, kind)), __builtin_bit_cast(vec8, w), (float4_t)(0.0f));
                        const float what = kind == 0 ? NAN : kind == 1 ? INFINITY : -INFINITY;
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            if (hit[r] > 0.0f) o[db][r] += what;
                    }
            }
        }
    };
    pass(std::false_type());
    float zero = 0.0f;
#pragma unroll
    for (int db = 0; db < D / 16; ++db)
#pragma unroll
        for (int r = 0; r < 4; ++r) zero = fmaf(o[db][r], 0.0f, zero);
    if (__any(zero != 0.0f || att_far<T>(m))) {
        pass(std::true_type());
        m += X::LIFT - X::LIFT_AGAIN;     // the other waves' unit
    }

    // the four waves' parts, through LDS: [wave][16 rows][D] sums, [wave][16] maxima and sums of a row; a quarter of each, so that four
    // finite ones end inside f32
    l += __shfl_xor(l, 16, 64);
    l += __shfl_xor(l, 32, 64);
    __syncthreads();
    constexpr int OLD = D + 4;
    float *so = (float *)smem, *sm = so + 4 * 16 * OLD, *sl = sm + 64;
#pragma unroll
    for (int db = 0; db < D / 16; ++db) *(floatx4 *)(so + (wave * 16 + l15) * OLD + 16 * db + 4 * quarter) = (floatx4){o[db][0], o[db][1], o[db][2], o[db][3]};
    if (quarter == 0) {
        sm[wave * 16 + l15] = m;
        sl[wave * 16 + l15] = l;
    }
    __syncthreads();
    for (int c = tid; c < p.rows * (D / 4); c += 256) {
        const int r = c / (D / 4), d4 = c % (D / 4) * 4;
        float top = -INFINITY;
#pragma unroll
        for (int w = 0; w < 4; ++w) top = fmaxf(top, sm[w * 16 + r]);
        const float base = top == -INFINITY ? 0.0f : top;
        float sum = 0.0f;
        floatx4 y = (floatx4)(0.0f);
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const float f = sm[w * 16 + r] == -INFINITY ? (sl[w * 16 + r] == 0.0f ? 0.0f : 0.25f) : 0.25f * att_exp2(sm[w * 16 + r] - base);
            sum = fmaf(f, sl[w * 16 + r], sum);
            const floatx4 x = *(const floatx4 *)(so + (w * 16 + r) * OLD + d4);      // zeros for a wave without keys
#pragma unroll
            for (int e = 0; e < 4; ++e) y[e] += att_weigh(f, x[e]);
        }
        const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
        sum *= 4.0f / (float)(1 << (int)X::LIFT);
        const int rt = p.by_group.div(r), rh = kvh * p.group + (r - rt * p.group);
        if (p.splits > 1) {
            const int64_t at = ((int64_t)pair * p.rows + r) * p.splits + split;
            *(floatx4 *)(p.part_o + at * D + d4) = (floatx4){y[0] * inv, y[1] * inv, y[2] * inv, y[3] * inv};
            if (d4 == 0) p.part_l[at] = sum == 0.0f ? -INFINITY : base + log2f(sum);
        } else {
            T *out = (T *)a.out + b * a.out_stride[0] + rt * a.out_stride[1] + rh * a.out_stride[2] + d4;
            *(uintx2 *)out = (uintx2){op_pack2(y[0] * inv, y[1] * inv, T()), op_pack2(y[2] * inv, y[3] * inv, T())};
            if (a.lse != nullptr && d4 == 0)
                a.lse[((int64_t)b * a.heads + rh) * a.q_tokens + rt] = sum == 0.0f ? -INFINITY : base * 0.6931471805599453f + logf(sum);
        }
    }
}

// ------------------------------------------------------------------------------------------------------------------
// Joins the parts of a row: one workgroup per row, D / 4 threads per part, 256 / (D / 4) parts at a time.
// Bound by latency (a few KB per row): eight loads per thread in flight, the first ones beside the search for the maximum (16 rows of 116
// parts 7.0 -> 4.8 us); slots without a part are skipped by the whole wave (1536 rows of 5 parts 4.8 us, 7.1 with idle slots).
template <typename T, int D>
__global__ __launch_bounds__(256) void attention_join_kernel(AttArgs p) {
    constexpr int TP = D / 4, G = 256 / TP;     // threads per part, parts at a time (D 96: 24 and 10, the last threads idle)
    __shared__ float red[G][D + 4];
    __shared__ float tops[4];
    const mibc_attention_args &a = p.a;
    const int tid = threadIdx.x;
    const int64_t r = blockIdx.x;
    const int pair = (int)(r / p.rows), row = (int)(r - (int64_t)pair * p.rows);
    const int b = p.by_kv.div(pair), kvh = pair - b * a.kv_heads;
    const int t = p.by_group.div(row), head = kvh * p.group + (row - t * p.group);
    const float *pl = p.part_l + r * p.splits;
    const float *po = p.part_o + r * p.splits * D;
    const int g = tid / TP, d4 = tid % TP * 4;
    floatx4 x[8];      // eight parts in flight per thread, the first ones while the maximum is found
    float w[8];
    auto fetch = [&](int first) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (first + i * G < p.splits) {
                const int s = first + i * G + g;
                const bool in = g < G && s < p.splits;
                x[i] = in ? *(const floatx4 *)(po + (int64_t)s * D + d4) : (floatx4)(0.0f);
                w[i] = in ? pl[s] : -INFINITY;
            }
    };
    fetch(0);
    float m = -INFINITY;
    for (int s = tid; s < p.splits; s += 256) m = fmaxf(m, pl[s]);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
    if ((tid & 63) == 0) tops[tid >> 6] = m;
    __syncthreads();
    m = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
    const float base = m == -INFINITY ? 0.0f : m;
    float sum = 0.0f;
    floatx4 y = (floatx4)(0.0f);
    for (int first = 0;;) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (first + i * G < p.splits) {
                const float f = att_exp2(w[i] - base) * 0x1p-8f;      // 255 finite parts end inside f32
                sum += f;
#pragma unroll
                for (int e = 0; e < 4; ++e) y[e] += att_weigh(f, x[i][e]);      // a part without keys holds zeros
            }
        first += 8 * G;
        if (first >= p.splits) break;
        fetch(first);
    }
    if (g < G) {
        *(floatx4 *)(&red[g][d4]) = y;
        if (d4 == 0) red[g][D] = sum;
    }
    __syncthreads();
    for (int d = tid; d < D; d += 256) {
        float v = 0.0f, n = 0.0f;
        for (int i = 0; i < G; ++i) {
            v += red[i][d];
            n += red[i][D];
        }
        const float inv = n == 0.0f ? 0.0f : 1.0f / n;
        ((T *)a.out + b * a.out_stride[0] + t * a.out_stride[1] + head * a.out_stride[2])[d] = (T)(v * inv);
        if (a.lse != nullptr && d == 0)
            a.lse[((int64_t)b * a.heads + head) * a.q_tokens + t] = n == 0.0f ? -INFINITY : base * 0.6931471805599453f + logf(n * 0x1p8f);
    }
}

template <typename T, int CAP, bool SLOPES>
static hipError_t att_one(hipStream_t s, const AttArgs &p, bool tokens) {
    // a launch holds less than 2^32 threads in x
    const unsigned x = p.groups < 1u << 20 ? p.groups : 1u << 20;
    const dim3 grid(x, (p.groups + x - 1) / x);
    constexpr int ROWS = 4 * 64 * ATT_D * 2, STEPS = 4 * 2 * 32 * ATT_D * 2, JOIN = 4 * 16 * (ATT_D + 4 + 2) * 4, TOKEN = STEPS > JOIN ? STEPS : JOIN;
#define ATT_GO(KERNEL, LDS)                                                             \
    do {                                                                                \
        MIBC_LDS_ATTR_ONCE(KERNEL, LDS);                                                \
        return op_launch(KERNEL, grid, 256, LDS, s, p);                                 \
    } while (0)
    if (tokens) ATT_GO((attention_token_kernel<T, ATT_D, CAP == ATT_NO_CAP ? ATT_NO_CAP : ATT_FAR, SLOPES>), TOKEN);
    ATT_GO((attention_kernel<T, ATT_D, CAP, SLOPES>), ROWS);
#undef ATT_GO
}
template <typename T>
static int att_launch(hipStream_t s, const AttArgs &p, bool tokens) {
#define ATT_S(CAP) (p.a.slopes ? att_one<T, CAP, true>(s, p, tokens) : att_one<T, CAP, false>(s, p, tokens))
    hipError_t rc = p.cap == ATT_FAR ? ATT_S(ATT_FAR) : p.cap == ATT_NEAR ? ATT_S(ATT_NEAR) : ATT_S(ATT_NO_CAP);
#undef ATT_S
    if (rc == hipSuccess && p.splits > 1)
        rc = op_launch(attention_join_kernel<T, ATT_D>, dim3((unsigned)((int64_t)p.pairs * p.rows)), 256, 0, s, p);
    return op_hip(rc, "attention");
}
#define ATT_CAT2(a, b) a##b
#define ATT_CAT(a, b) ATT_CAT2(a, b)
int ATT_CAT(mibc_att_launch_, ATT_D)(hipStream_t s, const AttArgs &p, bool tokens) {
    return p.a.type == MIBC_TYPE_F16 ? att_launch<half_t>(s, p, tokens) : att_launch<bf16_t>(s, p, tokens);
}
