// Pieces shared by the operators around the index (embedding.cu, quantize.cu, int8_matmul.cu, distill.cu): element types,
// several elements by one access, ids, checks of arguments.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "knn_common.cuh"

namespace cpb {
namespace op {

using knn::kFull;
using knn::smem_u32;

inline size_t type_bytes(int type) { return type == CPHNSW_B200_F32 ? 4 : 2; }
inline bool type_known(int type) { return type == CPHNSW_B200_F32 || type == CPHNSW_B200_F16 || type == CPHNSW_B200_BF16; }

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
template <class T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

template <int BYTES>
struct RawOf { using type = uint4; };
template <>
struct RawOf<1> { using type = uint8_t; };
template <>
struct RawOf<2> { using type = uint16_t; };
template <>
struct RawOf<4> { using type = uint32_t; };
template <>
struct RawOf<8> { using type = uint2; };

template <class T>
constexpr bool kIsBf16 = false;
template <>
constexpr bool kIsBf16<__nv_bfloat16> = true;

// E elements of T as accesses of up to 16 bytes (stores: of up to 32), the address a multiple of their size
template <class T, int E>
struct Pack {
    static constexpr int kBytes = E * int(sizeof(T)), kWord = kBytes < 16 ? kBytes : 16, kWords = kBytes / kWord;
    using Raw = typename RawOf<kWord>::type;
    union {
        Raw raw[kWords];
        T v[E];
    };
    __device__ __forceinline__ Pack() {}
    __device__ __forceinline__ void load(const T* p) {
#pragma unroll
        for (int i = 0; i < kWords; ++i) raw[i] = reinterpret_cast<const Raw*>(p)[i];
    }
    __device__ __forceinline__ void store(T* p) const {
        if constexpr (kBytes == 32) {  // (by one instruction: two of 16 bytes would each fill half of every sector)
            const uint32_t* w = reinterpret_cast<const uint32_t*>(raw);
            asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]),
                         "r"(w[6]), "r"(w[7])
                         : "memory");
        } else {
#pragma unroll
            for (int i = 0; i < kWords; ++i) reinterpret_cast<Raw*>(p)[i] = raw[i];
        }
    }
    __device__ __forceinline__ float get(int i) const { return to_float(v[i]); }
    __device__ __forceinline__ void set(int i, float f) { v[i] = from_float<T>(f); }
    // elements 2 i and 2 i + 1, rounded by one instruction where the type has one
    __device__ __forceinline__ void set2(int i, float a, float b) {
        if constexpr (sizeof(T) == 2) {
            if constexpr (kIsBf16<T>)
                reinterpret_cast<__nv_bfloat162*>(v)[i] = __floats2bfloat162_rn(a, b);
            else
                reinterpret_cast<__half2*>(v)[i] = __floats2half2_rn(a, b);
        } else {
            set(2 * i, a);
            set(2 * i + 1, b);
        }
    }
};

// two fp32 operations by one instruction
struct Two {
    float x, y;
};
__device__ __forceinline__ Two add(Two a, Two b) {
    Two r;
    asm("{\n\t.reg .b64 a, b;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tadd.rn.f32x2 a, a, b;\n\tmov.b64 {%0, %1}, a;\n\t}"
        : "=f"(r.x), "=f"(r.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return r;
}
__device__ __forceinline__ Two mul(Two a, Two b) {
    Two r;
    asm("{\n\t.reg .b64 a, b;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmul.rn.f32x2 a, a, b;\n\tmov.b64 {%0, %1}, a;\n\t}"
        : "=f"(r.x), "=f"(r.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return r;
}

__device__ __forceinline__ Two fma(Two a, Two b, Two c) {
    Two r;
    asm("{\n\t.reg .b64 a, b, c;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\tfma.rn.f32x2 a, a, b, c;\n\tmov.b64 {%0, %1}, a;\n\t}"
        : "=f"(r.x), "=f"(r.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return r;
}

// ids of 4 or 8 bytes; what lies outside [0, rows) is no row: kFull
struct Ids {
    const void* p;
    uint32_t bytes, rows;  // rows < 2^31
    __device__ __forceinline__ uint32_t at(uint64_t i) const {
        if (bytes == 8) {
            const int64_t v = __ldg(static_cast<const long long*>(p) + i);
            return v >= 0 && v < int64_t(rows) ? uint32_t(v) : kFull;
        }
        const uint32_t v = __ldg(static_cast<const unsigned int*>(p) + i);
        return v < rows ? v : kFull;
    }
};

// Elements of T that one access may take where all these addresses and byte strides are multiples of its size
struct Alignment {
    uint64_t bits = 0;
    Alignment& add(const void* p) {
        bits |= reinterpret_cast<uintptr_t>(p);
        return *this;
    }
    Alignment& add(uint64_t bytes) {
        bits |= bytes;
        return *this;
    }
    bool holds(uint64_t bytes) const { return bits % bytes == 0; }
};

// The word that bounded waits of the operators' kernels raise, one per device
int status_word(uint32_t** out);

constexpr int kMaxDevices = 64;
int sm_count(int* out);  // of the current device
int check_device();  // the current device is one this library runs on, its number below kMaxDevices
inline int invalid(const char* what) {
    set_error("%s", what);
    return CPHNSW_B200_E_INVALID;
}

#define CPB_OP_CHECK(ok, what) \
    do {                       \
        if (!(ok)) return cpb::op::invalid(what); \
    } while (0)

}  // namespace op
}  // namespace cpb
