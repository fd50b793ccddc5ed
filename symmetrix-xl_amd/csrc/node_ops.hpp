// What the node operators' sources share: value types, row access, checks of
// arguments and the C boundary.
#pragma once

#include <cstdint>
#include <new>
#include <stdexcept>
#include <string>
#include <type_traits>

#include "../../include/symmetrix_node_ops.h"
#include "device_common.hpp"

namespace smx {

void set_last_error(const std::string& message);  // evaluator.cpp

namespace node {

using bf16 = __bf16;
using f16 = _Float16;
using i64 = long long;

inline int size_of(int dtype) { return dtype == SMX_DTYPE_F32 ? 4 : 2; }

// f(T{}) with the value type of an SMX_DTYPE_* code
template <class F>
void with_dtype(int dtype, F&& f) {
    switch (dtype) {
        case SMX_DTYPE_F32: f(float{}); break;
        case SMX_DTYPE_BF16: f(bf16{}); break;
        case SMX_DTYPE_F16: f(f16{}); break;
        default: throw std::invalid_argument("unknown dtype code " + std::to_string(dtype));
    }
}

// N values as they lie in memory, aligned to one of them: global loads and
// stores of 16 bytes take any alignment on this target.
template <class T, int N>
struct __attribute__((packed, aligned(sizeof(T)))) Pack {
    T v[N];
};

// Eight values as the 32-bit words that hold them, so that 16-bit ones wait two in a register.
template <class T>
struct Eight {
    static constexpr int kWords = sizeof(T) * 2;
    std::uint32_t w[kWords];
    __device__ __forceinline__ float operator[](int i) const {
        if constexpr (sizeof(T) == 4) {
            return __uint_as_float(w[i]);
        } else if constexpr (std::is_same_v<T, bf16>) {
            return __uint_as_float(i % 2 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
        } else {
            return static_cast<float>(__builtin_bit_cast(f16, static_cast<std::uint16_t>(w[i / 2] >> (16 * (i % 2)))));
        }
    }
};

template <class T>
__device__ __forceinline__ std::uint32_t bits_of(T v) {
    if constexpr (sizeof(T) == 4)
        return __builtin_bit_cast(std::uint32_t, v);
    else
        return __builtin_bit_cast(std::uint16_t, v);
}

// Eight values from column c on (a multiple of eight), zeros past the end, in two steps, so that loads of several rows
// can be on their way together: a lane whose eight pass the row's end loads the row's last eight, like the others in
// one load without a branch of its own, and settle moves them to their places before they are used.  (With values
// loaded one by one in a branch, each row's loads waited for those of the row before: the embedding's gradient of 300,000
// rows of 447 FP32 took 254 us, of 448 137.)
template <class T>
__device__ __forceinline__ Eight<T> load_pack(const T* row, int c, int cols) {
    struct __attribute__((packed, aligned(sizeof(T)))) Words {
        std::uint32_t w[Eight<T>::kWords];
    };
    Eight<T> e;
    if (cols >= 8) {
        if (c < cols) {
            const Words p = *reinterpret_cast<const Words*>(row + (c + 8 <= cols ? c : cols - 8));
#pragma unroll
            for (int i = 0; i < Eight<T>::kWords; ++i) e.w[i] = p.w[i];
        } else {
#pragma unroll
            for (int i = 0; i < Eight<T>::kWords; ++i) e.w[i] = 0;
        }
        return e;
    }
    constexpr int kPer = 4 / sizeof(T);
#pragma unroll
    for (int i = 0; i < Eight<T>::kWords; ++i) {
        e.w[i] = c + kPer * i < cols ? bits_of(row[c + kPer * i]) : 0u;
        if constexpr (kPer == 2) e.w[i] |= c + 2 * i + 1 < cols ? bits_of(row[c + 2 * i + 1]) << 16 : 0u;
    }
    return e;
}

template <class T, int N>
__device__ __forceinline__ void settle(Eight<T> (&e)[N], int c, int cols) {
    if (cols < 8 || c >= cols || c + 8 <= cols) return;
    constexpr int kWords = Eight<T>::kWords, kPer = 4 / sizeof(T);
    const int by = -cols & 7;
#pragma unroll
    for (int n = 0; n < N; ++n) {
        std::uint32_t(&w)[kWords] = e[n].w;
        if (by & 4)
#pragma unroll
            for (int i = 0; i < kWords; ++i) w[i] = i + 4 / kPer < kWords ? w[(i + 4 / kPer) % kWords] : 0u;
        if (by & 2)
#pragma unroll
            for (int i = 0; i < kWords; ++i) w[i] = i + 2 / kPer < kWords ? w[(i + 2 / kPer) % kWords] : 0u;
        if (by & 1)
#pragma unroll
            for (int i = 0; i < kWords; ++i) {
                const std::uint32_t next = i + 1 < kWords ? w[(i + 1) % kWords] : 0u;
                w[i] = kPer == 1 ? next : w[i] >> 16 | next << 16;
            }
    }
}

template <class T>
__device__ __forceinline__ void settle(Eight<T>& e, int c, int cols) {
    settle(reinterpret_cast<Eight<T>(&)[1]>(e), c, cols);
}

template <class T>
__device__ __forceinline__ void load_eight(const T* row, int c, int cols, float (&v)[8]) {
    Eight<T> p = load_pack(row, c, cols);
    settle(p, c, cols);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = p[i];
}

// v, as another value to the compiler.  Where a whole store of neighbouring values and one value by value are two
// branches, the compiler makes the first value's store common to both and cuts the whole one into pieces.
__device__ __forceinline__ float apart(float v) {
    asm volatile("" : "+v"(v));
    return v;
}

// Eight values from column c on, up to the end.
template <class T>
__device__ __forceinline__ void store_eight(T* row, int c, int cols, const float (&v)[8]) {
    struct __attribute__((packed, aligned(sizeof(T)))) Words {
        std::uint32_t w[Eight<T>::kWords];
    };
    if (c + 8 <= cols) {
        Words p;
#pragma unroll
        for (int i = 0; i < Eight<T>::kWords; ++i) {
            if constexpr (sizeof(T) == 4)
                p.w[i] = bits_of(static_cast<T>(v[i]));
            else
                p.w[i] = bits_of(static_cast<T>(v[2 * i])) | bits_of(static_cast<T>(v[2 * i + 1])) << 16;
        }
        *reinterpret_cast<Words*>(row + c) = p;
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (c + i < cols) row[c + i] = static_cast<T>(apart(v[i]));
    }
}

// The sum of `count` parts, `hop` values apart, by a workgroup of 1024 for kJoined neighbouring values, whose first part is
// at `at`: 64 parts are read at once, so that the reads are few in a row (parts of 64 neighbouring values, 16 at once: 8.0 us
// for 512 parts of 2 x 999, 6.4 so).  The result is in the first kJoined lanes; the order is the same in every call.
constexpr int kJoined = 16;

__device__ __forceinline__ float sum_of_parts(const float* at, i64 hop, int count, bool in) {
    __shared__ float room[16][kJoined];
    const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
    float sum = 0.0f;
    if (in)
#pragma unroll 8
        for (int p = threadIdx.x / kJoined; p < count; p += 64) sum += at[p * hop];
    sum += __shfl_xor(sum, 16);
    sum += __shfl_xor(sum, 32);
    if (lane < kJoined) room[wave][lane] = sum;
    __syncthreads();
    sum = room[0][lane % kJoined];
#pragma unroll
    for (int w = 1; w < 16; ++w) sum += room[w][lane % kJoined];
    return sum;
}

inline void require(bool ok, const char* what) {
    if (!ok) throw std::invalid_argument(what);
}

inline bool aligned(const void* p, std::size_t to) { return reinterpret_cast<std::uintptr_t>(p) % to == 0; }

// checks one row array; an empty one needs no memory
inline void check_rows(const void* p, i64 stride, i64 rows, i64 channels, int dtype, const char* name) {
    if (rows > 0 && channels > 0 && !p) throw std::invalid_argument(std::string(name) + " is NULL");
    if (p && rows > 1 && stride < channels) throw std::invalid_argument(std::string(name) + ": the row stride is less than a row");
    if (!aligned(p, static_cast<std::size_t>(size_of(dtype)))) throw std::invalid_argument(std::string(name) + " is not aligned to its values");
}

inline void check_workspace(const void* p, i64 bytes, i64 needed) {
    if (needed == 0) return;
    if (!p || bytes < needed)
        throw std::invalid_argument("the workspace holds " + std::to_string(p ? bytes : 0) + " bytes, " + std::to_string(needed) +
                                    " are needed");
    require(aligned(p, 16), "the workspace is not 16-byte aligned");
}

template <class F>
int32_t guarded(F&& fn) noexcept {
    const auto failed = [](int32_t code, const char* what) {
        try {
            set_last_error(what);
        } catch (...) {  // no memory for the message
        }
        return code;
    };
    try {
        fn();
        return SMX_OK;
    } catch (const std::bad_alloc&) {
        return failed(SMX_ERR_OUT_OF_MEMORY, "out of memory");
    } catch (const std::domain_error& e) {
        return failed(SMX_ERR_UNSUPPORTED, e.what());
    } catch (const std::invalid_argument& e) {
        return failed(SMX_ERR_INVALID_ARGUMENT, e.what());
    } catch (const std::exception& e) {
        return failed(SMX_ERR_RUNTIME, e.what());
    } catch (...) {
        return failed(SMX_ERR_RUNTIME, "unknown error");
    }
}

// ---- 8-bit blocks ----

constexpr int kBlock = 128;

inline i64 block_stride(i64 cols) { return (cols + kBlock - 1) / kBlock * kBlock; }
inline i64 block_scale_stride(i64 cols) { return (block_stride(cols) / kBlock + 3) / 4 * 4; }

// The scale byte of a block whose largest finite magnitude is `top`: the
// least e >= -127 with top <= 448 * 2^e = 1.75 * 2^(e + 8), plus 127.
__device__ __forceinline__ int block_scale_byte(float top) {
    const unsigned bits = __float_as_uint(top);
    const int b = static_cast<int>(bits >> 23) - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
    return b < 0 ? 0 : b;
}

// 2^-(byte - 127), exact (bytes reach 247)
__device__ __forceinline__ float block_inverse_scale(int byte) {
    return __uint_as_float(static_cast<unsigned>(254 - byte) << 23);
}

// |v|, or 0 for an infinity or NaN
__device__ __forceinline__ float finite_magnitude(float v) {
    const float a = __builtin_fabsf(v);
    return a < __builtin_inff() ? a : 0.0f;
}

// an infinity becomes NaN: E4M3 has none
__device__ __forceinline__ float e4m3_input(float v, float inverse) {
    return __builtin_fabsf(v) < __builtin_inff() ? v * inverse : __builtin_nanf("");
}

__device__ __forceinline__ unsigned e4m3_four(float a, float b, float c, float d, float inverse) {
    int p = __builtin_amdgcn_cvt_pk_fp8_f32(e4m3_input(a, inverse), e4m3_input(b, inverse), 0, false);
    p = __builtin_amdgcn_cvt_pk_fp8_f32(e4m3_input(c, inverse), e4m3_input(d, inverse), p, true);
    return static_cast<unsigned>(p);
}

// max(v, v of the lane that the DPP control CTRL names)
template <int CTRL>
__device__ __forceinline__ float dpp_max(float v) {
    return fmaxf(v, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, false)));
}

// the largest of each row of 16 lanes, in all of them
__device__ __forceinline__ float row_max(float v) {
    v = dpp_max<0xb1>(v);
    v = dpp_max<0x4e>(v);
    v = dpp_max<0x141>(v);
    return dpp_max<0x140>(v);
}

__device__ __forceinline__ float top_of(const float (&v)[8]) {
    float top = finite_magnitude(v[0]);
#pragma unroll
    for (int i = 1; i < 8; ++i) top = fmaxf(top, finite_magnitude(v[i]));
    return top;
}

__device__ __forceinline__ uint2 e4m3_eight(const float (&v)[8], float inverse) {
    return make_uint2(e4m3_four(v[0], v[1], v[2], v[3], inverse), e4m3_four(v[4], v[5], v[6], v[7], inverse));
}

}  // namespace node
}  // namespace smx
