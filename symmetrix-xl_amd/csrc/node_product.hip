// Matrix products of E4M3 values with an E8M0 scale for each block of 128 values
// along the summed axis, and the kernels that bring matrices to that form.
//
// Two forms of the product, both with FP32 accumulators:
//   - 8-bit: v_mfma_scale_f32_16x16x128_f8f6f4 sums one block of 128 and applies both operands'
//     scales, powers of two, by itself.  Its adder aligns eight products to the largest of them
//     and drops what lies below 2^-13 of that one (measured: 2^16 + 127 products of 2^2 comes out
//     28 short, those of 2^4 exact), about 2^-18 of an output in rows of normal values.
//   - bf16: an E4M3 value times its scale is a bf16 value exactly (v_cvt_scalef32_pk_bf16_fp8), and
//     v_mfma_f32_16x16x32_bf16 sums as FP32 does, at half the rate.  (Values below 2^-126 count as zero there.)
// FP32 outputs take the bf16 form, so that their sums are FP32 sums.  16-bit outputs, which are rounded
// to 2^-9 or 2^-12 anyway, take the 8-bit form, but for short sums (up to 512), where a call is bound by its
// memory and the bf16 form costs nothing.
#include "node_ops.hpp"

namespace smx {
namespace node {
namespace {

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

constexpr i64 kShortSum = 512;

// Blocks along the rows: one wave per block.
template <class T>
__global__ void __launch_bounds__(256) k_quantize_rows(const T* __restrict__ x, i64 x_stride, i64 rows, i64 cols,
                                                       std::uint8_t* __restrict__ values,
                                                       std::uint8_t* __restrict__ scales, i64 pitch, i64 scale_pitch) {
    const int lane = threadIdx.x % 64;
    const i64 total = rows * scale_pitch;
    for (i64 b = static_cast<i64>(blockIdx.x) * 4 + threadIdx.x / 64; b < total; b += static_cast<i64>(gridDim.x) * 4) {
        const i64 r = b / scale_pitch, k = b % scale_pitch;
        if (k * kBlock >= pitch) {
            if (lane == 0) scales[b] = 0;
            continue;
        }
        const i64 c = k * kBlock + 2 * lane;
        const float v0 = c < cols ? static_cast<float>(x[r * x_stride + c]) : 0.0f;
        const float v1 = c + 1 < cols ? static_cast<float>(x[r * x_stride + c + 1]) : 0.0f;
        float top = fmaxf(finite_magnitude(v0), finite_magnitude(v1));
        for (int o = 32; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
        const int byte = block_scale_byte(top);
        const unsigned q = e4m3_four(v0, v1, 0.0f, 0.0f, block_inverse_scale(byte));
        *reinterpret_cast<std::uint16_t*>(values + r * pitch + c) = static_cast<std::uint16_t>(q);
        if (lane == 0) scales[b] = static_cast<std::uint8_t>(byte);
    }
}

// Blocks along the columns, stored as rows of the transpose: one wave per block.
template <class T>
__global__ void __launch_bounds__(256) k_quantize_columns(const T* __restrict__ x, i64 x_stride, i64 rows, i64 cols,
                                                          std::uint8_t* __restrict__ values,
                                                          std::uint8_t* __restrict__ scales, i64 pitch,
                                                          i64 scale_pitch) {
    const int lane = threadIdx.x % 64;
    const i64 total = cols * scale_pitch;
    for (i64 b = static_cast<i64>(blockIdx.x) * 4 + threadIdx.x / 64; b < total; b += static_cast<i64>(gridDim.x) * 4) {
        const i64 c = b / scale_pitch, k = b % scale_pitch;
        if (k * kBlock >= pitch) {
            if (lane == 0) scales[b] = 0;
            continue;
        }
        const i64 r = k * kBlock + 2 * lane;
        const float v0 = r < rows ? static_cast<float>(x[r * x_stride + c]) : 0.0f;
        const float v1 = r + 1 < rows ? static_cast<float>(x[(r + 1) * x_stride + c]) : 0.0f;
        float top = fmaxf(finite_magnitude(v0), finite_magnitude(v1));
        for (int o = 32; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
        const int byte = block_scale_byte(top);
        const unsigned q = e4m3_four(v0, v1, 0.0f, 0.0f, block_inverse_scale(byte));
        *reinterpret_cast<std::uint16_t*>(values + c * pitch + r) = static_cast<std::uint16_t>(q);
        if (lane == 0) scales[b] = static_cast<std::uint8_t>(byte);
    }
}

// The accumulators of a chain of MFMAs are read by other instructions right after it;
// eighteen wait states on every path into what follows (the 16x16x128 form takes
// eight passes), with the scheduler fenced on both sides.
__device__ __forceinline__ void mfma_settle() {
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_nop 8\n\ts_nop 8");
    __builtin_amdgcn_sched_barrier(0);
}

// Eight E4M3 values (two dwords) times a scale, as bf16.
__device__ __forceinline__ bf16x8 to_bf16(int lo, int hi, float scale) {
    const bf16x2 p[4] = {__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, false),
                         __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, true),
                         __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, false),
                         __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, true)};
    return __builtin_shufflevector(__builtin_shufflevector(p[0], p[1], 0, 1, 2, 3),
                                   __builtin_shufflevector(p[2], p[3], 0, 1, 2, 3), 0, 1, 2, 3, 4, 5, 6, 7);
}

// 2^(byte - 127) as a float
__device__ __forceinline__ float scale_of(int byte) {
    return byte ? __uint_as_float(static_cast<unsigned>(byte) << 23) : 0x1p-127f;
}

// 16 x 16 outputs a wave, operands straight from memory.  Lane l holds row
// l % 16 of both operands and bytes 32 (l / 16) on of the block (the order of
// k inside a block is the operands' own affair, as one scale covers it); the
// accumulator's lane l holds column l % 16 of rows 4 (l / 16) on, so with b as the first
// operand a lane's four values lie side by side in a row of the output.
template <class O, bool WIDE>
__global__ void __launch_bounds__(256) k_product_simple(const std::uint8_t* __restrict__ a,
                                                        const std::uint8_t* __restrict__ as,
                                                        const std::uint8_t* __restrict__ b,
                                                        const std::uint8_t* __restrict__ bs, i64 m, i64 n, i64 k,
                                                        i64 pitch, i64 scale_pitch, O* __restrict__ out,
                                                        i64 out_stride) {
    const int lane = threadIdx.x % 64;
    const i64 tiles_n = (n + 15) / 16, tiles = (m + 15) / 16 * tiles_n;
    const i64 tile = static_cast<i64>(blockIdx.x) * 4 + threadIdx.x / 64;
    if (tile >= tiles) return;
    const i64 i0 = tile / tiles_n * 16, j0 = tile % tiles_n * 16;
    const i64 i = i0 + lane % 16, j = j0 + lane % 16;
    const i64 ia = i < m ? i : m - 1, jb = j < n ? j : n - 1;
    const std::uint8_t* pa = a + ia * pitch + 32 * (lane / 16);
    const std::uint8_t* pb = b + jb * pitch + 32 * (lane / 16);
    acc4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
    for (i64 kb = 0; kb < pitch / kBlock; ++kb) {
        i32x8 va, vb;
        for (int h = 0; h < 2; ++h) {
            const i32x4 ha = *reinterpret_cast<const i32x4*>(pa + kb * kBlock + 16 * h);
            const i32x4 hb = *reinterpret_cast<const i32x4*>(pb + kb * kBlock + 16 * h);
            for (int q = 0; q < 4; ++q) va[4 * h + q] = ha[q], vb[4 * h + q] = hb[q];
        }
        const int sa = as[ia * scale_pitch + kb], sb = bs[jb * scale_pitch + kb];
        if constexpr (WIDE) {
            for (int q = 0; q < 4; ++q)
                acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(to_bf16(vb[2 * q], vb[2 * q + 1], scale_of(sb)),
                                                              to_bf16(va[2 * q], va[2 * q + 1], scale_of(sa)), acc, 0, 0, 0);
        } else {
            acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(vb, va, acc, 0, 0, 0, sb, 0, sa);
        }
    }
    mfma_settle();
    if (i >= m) return;
    for (int v = 0; v < 4; ++v) {
        const i64 col = j0 + 4 * (lane / 16) + v;
        if (col < n) out[i * out_stride + col] = static_cast<O>(acc[v]);
    }
}

void check_sizes(i64 m, i64 n, i64 k) {
    require(m >= 0 && m < (1LL << 31) && n >= 0 && n < (1LL << 31) && k >= 0 && k < (1LL << 31),
            "sizes must be in [0, 2^31)");
}

void check_blocks(const void* values, const void* scales, i64 rows, i64 cols, const char* name) {
    if (rows == 0 || cols == 0) return;
    if (!values || !scales) throw std::invalid_argument(std::string(name) + " is NULL");
    if (!aligned(values, 16) || !aligned(scales, 16))
        throw std::invalid_argument(std::string(name) + ": 8-bit blocks must be 16-byte aligned");
}

template <class T>
void launch_quantize(const void* x, i64 x_stride, i64 rows, i64 cols, std::uint8_t* values, std::uint8_t* scales,
                     std::uint8_t* values_t, std::uint8_t* scales_t, hipStream_t stream) {
    const auto grid = [](i64 blocks) { return static_cast<unsigned>(blocks < 4 * 65536 ? (blocks + 3) / 4 : 65536); };
    if (values && rows > 0 && cols > 0) {
        const i64 pitch = block_stride(cols), scale_pitch = block_scale_stride(cols);
        k_quantize_rows<T><<<grid(rows * scale_pitch), 256, 0, stream>>>(static_cast<const T*>(x), x_stride, rows, cols,
                                                                       values, scales, pitch, scale_pitch);
        SMX_LAUNCH_CHECK("k_quantize_rows");
    }
    if (values_t && rows > 0 && cols > 0) {
        const i64 pitch = block_stride(rows), scale_pitch = block_scale_stride(rows);
        k_quantize_columns<T><<<grid(cols * scale_pitch), 256, 0, stream>>>(static_cast<const T*>(x), x_stride, rows,
                                                                          cols, values_t, scales_t, pitch, scale_pitch);
        SMX_LAUNCH_CHECK("k_quantize_columns");
    }
}

template <class O>
void launch_product(const std::uint8_t* a, const std::uint8_t* as, const std::uint8_t* b, const std::uint8_t* bs, i64 m,
                    i64 n, i64 k, O* out, i64 out_stride, hipStream_t stream) {
    const i64 tiles = (m + 15) / 16 * ((n + 15) / 16);
    const bool wide = sizeof(O) == 4 || k <= kShortSum;
    (wide ? k_product_simple<O, true> : k_product_simple<O, false>)<<<blocks_for(tiles, 4), 256, 0, stream>>>(
        a, as, b, bs, m, n, k, block_stride(k), block_scale_stride(k), out, out_stride);
    SMX_LAUNCH_CHECK("k_product_simple");
}

}  // namespace
}  // namespace node
}  // namespace smx

using namespace smx;
using namespace smx::node;

extern "C" {

int64_t smx_block_stride(int64_t cols) { return cols > 0 ? block_stride(cols) : 0; }
int64_t smx_block_scale_stride(int64_t cols) { return cols > 0 ? block_scale_stride(cols) : 0; }

int32_t smx_block_quantize(const void* x, int64_t x_stride, int32_t dtype, int64_t rows, int64_t cols, uint8_t* values,
                           uint8_t* scales, uint8_t* values_t, uint8_t* scales_t, void* stream) {
    return guarded([&] {
        check_sizes(rows, cols, 0);
        require(dtype >= SMX_DTYPE_F32 && dtype <= SMX_DTYPE_F16, "unknown dtype code");
        check_rows(x, x_stride, rows, cols, dtype, "x");
        require(!values == !scales && !values_t == !scales_t, "values and scales go together");
        require(values || values_t || rows == 0 || cols == 0, "no output is asked for");
        if (values) check_blocks(values, scales, rows, cols, "values");
        if (values_t) check_blocks(values_t, scales_t, rows, cols, "values_t");
        with_dtype(dtype, [&](auto t) {
            launch_quantize<decltype(t)>(x, x_stride, rows, cols, values, scales, values_t, scales_t,
                                         static_cast<hipStream_t>(stream));
        });
    });
}

int64_t smx_block_product_workspace(int64_t, int64_t, int64_t) { return 0; }

int32_t smx_block_product(const uint8_t* a_values, const uint8_t* a_scales, const uint8_t* b_values,
                          const uint8_t* b_scales, int64_t m, int64_t n, int64_t k, int32_t dtype, void* out,
                          int64_t out_stride, void* workspace, int64_t workspace_bytes, void* stream) {
    return guarded([&] {
        check_sizes(m, n, k);
        require(dtype >= SMX_DTYPE_F32 && dtype <= SMX_DTYPE_F16, "unknown dtype code");
        check_blocks(a_values, a_scales, m, k, "a");
        check_blocks(b_values, b_scales, n, k, "b");
        check_rows(out, out_stride, m, n, dtype, "out");
        check_workspace(workspace, workspace_bytes, smx_block_product_workspace(m, n, k));
        if (m == 0 || n == 0) return;
        with_dtype(dtype, [&](auto o) {
            using O = decltype(o);
            launch_product<O>(a_values, a_scales, b_values, b_scales, m, n, k, static_cast<O*>(out), out_stride,
                              static_cast<hipStream_t>(stream));
        });
    });
}

int64_t smx_block_linear_workspace(int64_t m, int64_t n, int64_t k) {
    if (m <= 0 || n <= 0 || k <= 0) return 0;
    return m * block_stride(k) + (m * block_scale_stride(k) + 15) / 16 * 16;
}

int32_t smx_block_linear(const void* x, int64_t x_stride, int32_t dtype, const uint8_t* w_values,
                         const uint8_t* w_scales, int64_t m, int64_t n, int64_t k, int32_t out_dtype, void* out,
                         int64_t out_stride, void* workspace, int64_t workspace_bytes, void* stream) {
    return guarded([&] {
        check_sizes(m, n, k);
        require(dtype >= SMX_DTYPE_F32 && dtype <= SMX_DTYPE_F16, "unknown dtype code");
        require(out_dtype >= SMX_DTYPE_F32 && out_dtype <= SMX_DTYPE_F16, "unknown dtype code");
        check_rows(x, x_stride, m, k, dtype, "x");
        check_blocks(w_values, w_scales, n, k, "w");
        check_rows(out, out_stride, m, n, out_dtype, "out");
        check_workspace(workspace, workspace_bytes, smx_block_linear_workspace(m, n, k));
        if (m == 0 || n == 0) return;
        auto* const values = static_cast<std::uint8_t*>(workspace);
        std::uint8_t* const scales = k > 0 ? values + m * block_stride(k) : nullptr;
        if (k > 0)
            with_dtype(dtype, [&](auto t) {
                launch_quantize<decltype(t)>(x, x_stride, m, k, values, scales, nullptr, nullptr,
                                             static_cast<hipStream_t>(stream));
            });
        with_dtype(out_dtype, [&](auto o) {
            using O = decltype(o);
            launch_product<O>(values, scales, w_values, w_scales, m, n, k, static_cast<O*>(out), out_stride,
                              static_cast<hipStream_t>(stream));
        });
    });
}

}  // extern "C"
