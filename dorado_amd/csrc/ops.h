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
    mibc_gerr() = std::string(what) + ": " + hipGetErrorString(rc);
    return MIBC_ERR_HIP;
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
