// Products in tiles, shared by the products by kind of row and the products in 8-bit integers: operands go to LDS in steps of
// 128 bytes of the summed axis, and matrix instructions take them from there.
//
// An operand lies in one of two ways: its summed axis along the rows (Rows: x and the weights of a forward product) or
// across them (Columns: the weights of a gradient by x, both operands of one by the weights).  A step of V 16-bit values of the summed
// axis of B outer indices is B * V * 2 bytes of LDS either way, in pieces of 16 bytes:
//   Rows     [B][V / 8 pieces], a row's pieces permuted by the row's number, so that the 16 rows that a fragment read meets at once
//            lie in different banks;
//   Columns  [V][B / 8 pieces], 16 columns together, these permuted by the row, so that the rows that a transposing read
//            (ds_read_b64_tr_b16: four rows of 16 columns for 16 lanes) meets at once do.
// Rows that are aligned to 16 bytes and as long as whole pieces go from memory to LDS without registers; a piece that is not there (past
// the summed axis' end) is read from a place of zeros, so both operands are zero there and infinities outside a sum stay
// outside.  Other rows, and FP32 ones, whose parts are formed on the way, go through registers.
//
// The order of the summed axis inside a step is the operands' own affair, as long as it is one: piece p holds values 8 p .. 8 p + 7,
// instruction q takes pieces 4 q .. 4 q + 3, lane group l / 16 the piece 4 q + l / 16.
#pragma once

#include <type_traits>
#include <utility>

#include "node_ops.hpp"

namespace smx {
namespace node {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

enum class Lie { Rows, Columns };

constexpr int kStepBytes = 128;
constexpr int kComputeUnits = 256;

// where pieces that are not there are read from
static __device__ const uint4 kNothing[1] = {};

// sixteen bytes of global memory (a choice of two places is one of any address space to the compiler)
__device__ __forceinline__ i32x4 load_sixteen(const void* at) {
    return *(const __attribute__((address_space(1))) i32x4*)(reinterpret_cast<std::uintptr_t>(at));
}

// 1 KB of LDS at byte lds + OFFSET (the wave's own, uniform) from 64 lanes' 16 bytes: memory to LDS without registers.  The compiler
// does not count it: arrived().
template <int OFFSET>
__device__ __forceinline__ void fetch(const void* at, unsigned lds) {
    asm volatile("s_add_u32 m0, %0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" : : "s"(lds), "v"(at), "n"(OFFSET) : "memory", "scc");
}
// f(0), ..., f(N - 1) with the number as a constant
template <int N, class F>
__device__ __forceinline__ void each_of(F&& f) {
    [&]<int... I>(std::integer_sequence<int, I...>) __attribute__((always_inline)) {
        (f(std::integral_constant<int, I>{}), ...);
    }(std::make_integer_sequence<int, N>{});
}
__device__ __forceinline__ void arrived() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

// The accumulators of a chain of MFMAs are read by other instructions right after it; eighteen wait states on every path
// into what follows, with the scheduler fenced on both sides.
__device__ __forceinline__ void settle_products() {
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_nop 8\n\ts_nop 8");
    __builtin_amdgcn_sched_barrier(0);
}

// Sixteen bytes of a row from value c on (c a multiple of what they hold), zeros past its end, at any alignment: a piece that
// passes the end loads the row's last sixteen bytes, and settle_piece moves them to their places.
template <class T>
__device__ __forceinline__ i32x4 load_piece(const T* row, i64 c, i64 cols) {
    constexpr int kPer = 16 / sizeof(T);
    struct __attribute__((packed, aligned(sizeof(T)))) Words {
        i32x4 w;
    };
    if (cols >= kPer) {
        if (c >= cols) return i32x4{0, 0, 0, 0};
        return reinterpret_cast<const Words*>(row + (c + kPer <= cols ? c : cols - kPer))->w;
    }
    i32x4 w{0, 0, 0, 0};
    constexpr int kHalf = 4 / sizeof(T);
#pragma unroll
    for (int i = 0; i < kPer; ++i)
        if (c + i < cols) w[i / kHalf] |= static_cast<int>(bits_of(row[c + i]) << (i % kHalf * 8 * sizeof(T)));
    return w;
}

template <class T>
__device__ __forceinline__ i32x4 settle_piece(i32x4 w, i64 c, i64 cols) {
    constexpr int kPer = 16 / sizeof(T);
    if (cols < kPer || c >= cols || c + kPer <= cols) return w;
    const int by = static_cast<int>(c + kPer - cols) * static_cast<int>(sizeof(T));  // bytes to move down
    if (by & 8) w = i32x4{w[2], w[3], 0, 0};
    if (by & 4) w = i32x4{w[1], w[2], w[3], 0};
    if constexpr (sizeof(T) == 2) {
        if (by & 2) {
            const auto half = [](int lo, int hi) {
                return static_cast<int>(static_cast<unsigned>(lo) >> 16 | static_cast<unsigned>(hi) << 16);
            };
            w = i32x4{half(w[0], w[1]), half(w[1], w[2]), half(w[2], w[3]), half(w[3], 0)};
        }
    }
    return w;
}

// ---- an operand's step in LDS ----

// VALUES 16-bit values (or pairs of bytes) of the summed axis of B outer indices.
template <Lie L, int B, int VALUES>
struct Step {
    static constexpr int kBytes = B * VALUES * 2, kPieces = kBytes / 16;
    static constexpr int kRowPieces = L == Lie::Rows ? VALUES / 8 : B / 8;

    __device__ __forceinline__ static int turned(int row) {
        // Sixteen lanes of a read meet at once, not in order: 0-3, 12-15 of the first sixteen and 4-11 of the next (so conflicts were
        // counted at rows of four pieces: 138 million cycles of 377 with row / 4 % 4 for them).  0, 2, 3, 1 parts these.
        if constexpr (L == Lie::Rows && VALUES == 32) return 0x78 >> row / 4 % 4 * 2 & 3;
        if constexpr (L == Lie::Rows) return row / (128 / VALUES) % (VALUES / 8);
        return (row / 8 * 4 + row % 4) & (B / 16 - 1);
    }
    // the row and the piece of it that lie at piece e of the step
    __device__ __forceinline__ static int row_at(int e) { return e / kRowPieces; }
    __device__ __forceinline__ static int piece_at(int e) {
        const int p = e % kRowPieces, t = turned(e / kRowPieces);
        if constexpr (L == Lie::Rows) return p ^ t;
        return ((p / 2) ^ t) * 2 + p % 2;
    }
    // the byte at which half `half` of piece p of a row lies
    __device__ __forceinline__ static int place(int row, int p, int half) {
        if constexpr (L == Lie::Rows) return (row * kRowPieces + (p ^ turned(row))) * 16 + half * 8;
        return (row * kRowPieces + (((p / 2) ^ turned(row)) * 2 + p % 2)) * 16 + half * 8;
    }
    // 16 outer indices from `outer` (a multiple of 16) on, values 32 q .. 32 q + 31: what instruction q takes of lane l, whose
    // outer index is l % 16
    __device__ __forceinline__ static i32x4 read(const std::uint8_t* tile, int outer, int q, int lane) {
        if constexpr (L == Lie::Rows) {
            return *reinterpret_cast<const i32x4*>(tile + outer * VALUES * 2 + lane % 16 * VALUES * 2 +
                                                   ((lane / 16 ^ turned(lane % 16)) ^ 4 * q) * 16);
        } else {
            using At = __attribute__((address_space(3))) s16x4*;
            typedef int i32x2 __attribute__((ext_vector_type(2)));
            constexpr int kPitch = B * 2;
            const std::uint8_t* const at = tile + (8 * (lane / 16) + lane % 16 / 4) * kPitch +
                                           ((outer / 16) ^ (lane / 4 & (B / 16 - 1))) * 32 + lane % 4 * 8;
            i32x2 h[2];
#pragma unroll
            for (int k = 0; k < 2; ++k)
                h[k] = __builtin_bit_cast(i32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((At)(at + (32 * q + 4 * k) * kPitch)));
            return __builtin_shufflevector(h[0], h[1], 0, 1, 2, 3);
        }
    }
};

// ---- the matrix instructions by type: 64 bytes of the summed axis ----

template <class T>
struct Multiply;
template <>
struct Multiply<bf16> {
    using Sum = acc4;
    __device__ __forceinline__ static acc4 add(i32x4 b, i32x4 a, acc4 acc) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, b), __builtin_bit_cast(bf16x8, a), acc, 0, 0, 0);
    }
};
template <>
struct Multiply<f16> {
    using Sum = acc4;
    __device__ __forceinline__ static acc4 add(i32x4 b, i32x4 a, acc4 acc) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, b), __builtin_bit_cast(f16x8, a), acc, 0, 0, 0);
    }
};
template <>
struct Multiply<std::int8_t> {
    using Sum = i32x4;
    __device__ __forceinline__ static i32x4 add(i32x4 b, i32x4 a, i32x4 acc) {
        return __builtin_amdgcn_mfma_i32_16x16x64_i8(b, a, acc, 0, 0, 0);
    }
};
// FP32: three bf16 parts of each operand, the smallest products first (device_common.hpp): FP32's precision at a sixth of
// bf16's rate, where the FP32 matrix instructions have a sixteenth.
struct Parts {
    i32x4 part[3];
};
__device__ __forceinline__ acc4 add_parts(const Parts& b, const Parts& a, acc4 acc) {
    constexpr int pb[6] = {0, 2, 1, 0, 1, 0}, pa[6] = {2, 0, 1, 1, 0, 0};
#pragma unroll
    for (int q = 0; q < 6; ++q) acc = Multiply<bf16>::add(b.part[pb[q]], a.part[pa[q]], acc);
    return acc;
}

// Four FP32 values as three bf16 parts of each: what split_operand (device_common.hpp) does with eight.
struct FourParts {
    uint2 part[3];
};
__device__ __forceinline__ FourParts split_four(i32x4 w) {
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    FourParts o;
    float x[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = __int_as_float(w[i]);
#pragma unroll
    for (int p = 0; p < 3; ++p) {
        unsigned bits[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const float big = p == 0 ? kSplitMax : kSplitMax2;
            const f32x2 v = p == 2 ? f32x2{x[2 * h], x[2 * h + 1]}
                                   : f32x2{__builtin_amdgcn_fmed3f(x[2 * h], -big, big), __builtin_amdgcn_fmed3f(x[2 * h + 1], -big, big)};
            bits[h] = __builtin_bit_cast(unsigned, __builtin_convertvector(v, bf16x2));
            if (p < 2) {
                x[2 * h] -= __uint_as_float(bits[h] << 16);
                x[2 * h + 1] -= __uint_as_float(bits[h] & 0xffff0000u);
            }
        }
        o.part[p] = make_uint2(bits[0], bits[1]);
    }
    return o;
}

// ---- up to sixteen rows ----

template <class T>
struct SumType {
    using type = typename Multiply<T>::Sum;
};
template <>
struct SumType<float> {
    using type = acc4;
};
template <class T>
using SumOf = typename SumType<T>::type;

// Where the waves of few_rows meet.
template <class T, int NF, int KS>
struct FewRoom {
    SumOf<T> v[KS][NF][64];
};

// Sixteen rows of a times 16 NF rows of b by KS waves, every KS-th step each, joined in LDS: where the bytes of b are all of it, they
// go straight to registers, kAhead steps of them under way at once.  `a` and `b`: the rows of the lane (l % 16).  The sums of the
// waves are left in the room; joined() adds up fragment g's (lane l: column l % 16, four rows of b from 4 (l / 16) on).
template <class T, bool DIRECT, int NF, int KS>
__device__ __forceinline__ void few_rows(const T* a, const T* const (&b)[NF], int k, FewRoom<T, NF, KS>& room) {
    using Sum = SumOf<T>;
    constexpr int kAhead = 4, kValues = kStepBytes / static_cast<int>(sizeof(T)), kPer = 16 / static_cast<int>(sizeof(T));
    // (a wave's branches have to be the whole wave's to the compiler too: matrix instructions run for all lanes)
    const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const int steps = (k + kValues - 1) / kValues;
    const auto load = [&](const T* row, int c) {
        if constexpr (DIRECT)
            return load_sixteen(c < k ? static_cast<const void*>(row + c) : kNothing);
        else
            return load_piece(row, c, k);
    };
    Sum acc[NF];
#pragma unroll
    for (int g = 0; g < NF; ++g) acc[g] = Sum{0, 0, 0, 0};
    for (int s0 = wave; s0 < steps; s0 += KS * kAhead) {
        i32x4 wb[kAhead][NF][2], wa[kAhead][2];
#pragma unroll
        for (int q = 0; q < kAhead; ++q) {
            const int s = s0 + q * KS < steps ? s0 + q * KS : s0;  // (a step read twice is used once)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int c = s * kValues + (lane / 16 + 4 * h) * kPer;
                wa[q][h] = load(a, c);
#pragma unroll
                for (int g = 0; g < NF; ++g) wb[q][g][h] = load(b[g], c);
            }
        }
#pragma unroll
        for (int q = 0; q < kAhead; ++q) {
            if (s0 + q * KS >= steps) break;
            if constexpr (!DIRECT)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int c = (s0 + q * KS) * kValues + (lane / 16 + 4 * h) * kPer;
                    wa[q][h] = settle_piece<T>(wa[q][h], c, k);
#pragma unroll
                    for (int g = 0; g < NF; ++g) wb[q][g][h] = settle_piece<T>(wb[q][g][h], c, k);
                }
            if constexpr (sizeof(T) == 4) {
                const auto parts = [](i32x4 lo, i32x4 hi) {
                    typedef int i32x8 __attribute__((ext_vector_type(8)));
                    const i32x8 both = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
                    return split_operand(__builtin_bit_cast(f32x8, both));
                };
                const SplitOperand va = parts(wa[q][0], wa[q][1]);
#pragma unroll
                for (int g = 0; g < NF; ++g) acc[g] = split_product(parts(wb[q][g][0], wb[q][g][1]), va, acc[g]);
            } else {
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int g = 0; g < NF; ++g) acc[g] = Multiply<T>::add(wb[q][g][h], wa[q][h], acc[g]);
            }
            settle_products();  // (the next step is conditional)
        }
    }
    settle_products();
#pragma unroll
    for (int g = 0; g < NF; ++g) room.v[wave][g][lane] = acc[g];
    __syncthreads();
}

template <class T, int NF, int KS>
__device__ __forceinline__ SumOf<T> joined(const FewRoom<T, NF, KS>& room, int g) {
    const int lane = threadIdx.x % 64;
    SumOf<T> sum = room.v[0][g][lane];
#pragma unroll
    for (int w = 1; w < KS; ++w) sum += room.v[w][g][lane];
    return sum;
}

}  // namespace node
}  // namespace smx
