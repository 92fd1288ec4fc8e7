// dorado_amd/csrc/ops.h — shared by the transformer-layer operators (ops_norm.hip, ops_rope.hip, ops_attention.hip): element types,
// the launch on a caller's device and stream.  Not part of the public ABI (that is include/mibc.h).
#pragma once
#include "../../include/mibc.h"
#include "common.h"

#include <string>

std::string &mibc_gerr();   // text behind mibc_last_error(NULL), per thread (engine.hip)

typedef __bf16 bf16_t;
typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef unsigned uintx2 __attribute__((ext_vector_type(2)));
typedef unsigned uintx4 __attribute__((ext_vector_type(4)));
typedef float float2_ops __attribute__((ext_vector_type(2)));
typedef bf16_t bf16x2_t __attribute__((ext_vector_type(2)));

static inline int op_refuse(int code, const std::string &what) {
    mibc_gerr() = what;
    return code;
}

// Makes `device` current for the launches of one call and puts the caller's device back.
struct OpDevice {
    int before = -1, want;
    hipError_t rc;
    explicit OpDevice(int device) : want(device) {
        rc = hipGetDevice(&before);
        if (rc == hipSuccess && before != want) rc = hipSetDevice(want);
    }
    ~OpDevice() {
        if (rc == hipSuccess && before != want) (void)hipSetDevice(before);
    }
};
static inline int op_hip(hipError_t rc, const char *what) {
    if (rc == hipSuccess) return MIBC_OK;
    (void)hipGetLastError();      // reported here, not by the caller's next call as well
    mibc_gerr() = std::string(what) + ": " + hipGetErrorString(rc);
    return MIBC_ERR_HIP;
}
// The launch's own status: the thread's last error may be an older one of the program's
template <typename A>
static inline hipError_t op_launch(void (*kernel)(A), dim3 grid, unsigned threads, unsigned lds, hipStream_t s, const A &args) {
    void *list[1] = {(void *)&args};
    return hipLaunchKernel((const void *)kernel, grid, dim3(threads), list, lds, s);
}

// The memory of an operand: runs of bytes at base + sum i_d stride_d, i_d < size_d.  A stride of 0 is a broadcast dimension.
struct OpSpan {
    uintptr_t base, end;      // equal where there is nothing
    int64_t run, size[3], stride[3];
};
static inline OpSpan op_span(const void *base, int64_t run, int64_t n0 = 1, int64_t s0 = 0, int64_t n1 = 1, int64_t s1 = 0, int64_t n2 = 1, int64_t s2 = 0) {
    OpSpan s = {(uintptr_t)base, (uintptr_t)base, run, {n0, n1, n2}, {s0, s1, s2}};
    if (base == nullptr || n0 == 0 || n1 == 0 || n2 == 0) return s;
    // no operand reaches beyond 2^63 bytes
    s.end += run + (n0 > 1 ? (n0 - 1) * s0 : 0) + (n1 > 1 ? (n1 - 1) * s1 : 0) + (n2 > 1 ? (n2 - 1) * s2 : 0);
    return s;
}
static inline bool op_same(const OpSpan &a, const OpSpan &b) {
    bool same = a.base == b.base && a.run == b.run;
    for (int d = 0; d < 3; ++d) same = same && a.size[d] == b.size[d] && (a.size[d] <= 1 || a.stride[d] == b.stride[d]);
    return same;
}
// Whether no byte of an output is written twice: every stride steps over all that the smaller ones reach, as in any view of a dense buffer.
static inline bool op_plain(const OpSpan &s) {
    for (int d = 0; d < 3; ++d) {
        if (s.size[d] <= 1) continue;
        int64_t n = s.run;
        for (int e = 0; e < 3; ++e)
            if (e != d && s.size[e] > 1 && (s.stride[e] < s.stride[d] || (s.stride[e] == s.stride[d] && e > d))) n += (s.size[e] - 1) * s.stride[e];
        if (s.stride[d] < n) return false;
    }
    return true;
}
// Whether two operands share no byte.  Either their ends show it, or the strides from some size on are all multiples of an M, and what
// the smaller strides reach of each lies apart within M (columns of one packed buffer, heads or rows dealt to two tensors).  False for
// what neither shows
static inline bool op_apart(const OpSpan &a, const OpSpan &b) {
    if (a.end <= b.base || b.end <= a.base || a.end == a.base || b.end == b.base) return true;
    const OpSpan *const both[2] = {&a, &b};
    auto reach = [](const OpSpan &s, int64_t below) {     // bytes from the base to the end, strides below that limit only
        int64_t n = s.run;
        for (int d = 0; d < 3; ++d)
            if (s.stride[d] < below && s.size[d] > 1) n += (s.size[d] - 1) * s.stride[d];
        return n;
    };
    const int64_t from = (int64_t)(b.base - a.base);
    for (const OpSpan *s : both)
        for (int d = 0; d < 3; ++d) {
            const int64_t least = s->stride[d];
            if (s->size[d] <= 1 || least == 0) continue;
            int64_t m = 0;
            for (const OpSpan *t : both)
                for (int e = 0; e < 3; ++e)
                    if (t->size[e] > 1 && t->stride[e] >= least)
                        for (int64_t x = t->stride[e]; x != 0;) {
                            const int64_t rest = m % x;
                            m = x;
                            x = rest;
                        }
            const int64_t off = (from % m + m) % m;
            if (off >= reach(a, least) && off <= m - reach(b, least)) return true;
        }
    return false;
}

static inline int op_type_bytes(int type) { return type == MIBC_TYPE_F32 ? 4 : (type == MIBC_TYPE_I8 || type == MIBC_TYPE_E4M3) ? 1 : 2; }
static inline bool op_aligned(const void *p, unsigned bytes) { return ((uintptr_t)p & (bytes - 1)) == 0; }

// eight consecutive elements <-> f32; the 16-bit ones round to nearest even (v_cvt_pk_*_f32).  ANY: at any address (global memory
// takes 16-byte accesses there too, at about two thirds of the rate)
template <typename V, bool ANY>
__device__ __forceinline__ V op_get(const void *p) {
    if (!ANY) return *(const V *)p;
    V v;
    __builtin_memcpy(&v, p, sizeof(V));
    return v;
}
template <typename V, bool ANY>
__device__ __forceinline__ void op_put(void *p, V v) {
    if (!ANY) *(V *)p = v;
    else __builtin_memcpy(p, &v, sizeof(V));
}
template <bool ANY = false>
__device__ __forceinline__ void op_load8(const half_t *p, float v[8]) {
    const half8_t x = op_get<half8_t, ANY>(p);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = (float)x[i];
}
template <bool ANY = false>
__device__ __forceinline__ void op_load8(const bf16_t *p, float v[8]) {
    const uintx4 x = op_get<uintx4, ANY>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[2 * i] = __uint_as_float(x[i] << 16);
        v[2 * i + 1] = __uint_as_float(x[i] & 0xffff0000u);
    }
}
template <bool ANY = false>
__device__ __forceinline__ void op_load8(const float *p, float v[8]) {
    const floatx4 a = op_get<floatx4, ANY>(p), b = op_get<floatx4, ANY>(p + 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[i] = a[i];
        v[4 + i] = b[i];
    }
}
__device__ __forceinline__ unsigned op_pack2(float a, float b, half_t) {
    const float2_ops x = {a, b};
    return __builtin_bit_cast(unsigned, __builtin_convertvector(x, half2_t));
}
__device__ __forceinline__ unsigned op_pack2(float a, float b, bf16_t) {
    const float2_ops x = {a, b};
    return __builtin_bit_cast(unsigned, __builtin_convertvector(x, bf16x2_t));
}
template <typename T, bool ANY = false>
__device__ __forceinline__ void op_store8(T *p, const float v[8]) {
    if constexpr (sizeof(T) == 4) {
        op_put<floatx4, ANY>(p, (floatx4){v[0], v[1], v[2], v[3]});
        op_put<floatx4, ANY>(p + 4, (floatx4){v[4], v[5], v[6], v[7]});
    } else {
        uintx4 x;
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = op_pack2(v[2 * i], v[2 * i + 1], T());
        op_put<uintx4, ANY>(p, x);
    }
}
