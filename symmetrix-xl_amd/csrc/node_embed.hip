// Species embedding: scaled rows of a table by type, and the gradient of the
// table, summed over the atoms of each type.
#include "node_ops.hpp"

namespace smx {
namespace node {
namespace {

// The type of atom t, or -1 where it is none of the table's.
template <class I>
__device__ __forceinline__ int type_of(const I* types, i64 t, i64 num_types) {
    const I z = types[t];
    return z >= 0 && static_cast<i64>(z) < num_types ? static_cast<int>(z) : -1;
}

// One thread per value.
template <class T, class I>
__global__ void __launch_bounds__(256) k_embed(const I* __restrict__ types, i64 tokens, const T* __restrict__ table,
                                               i64 table_stride, i64 num_types, i64 channels, float scale,
                                               T* __restrict__ out, i64 out_stride) {
    for (i64 t = blockIdx.x; t < tokens; t += gridDim.x) {
        const int z = type_of(types, t, num_types);
        for (i64 c = threadIdx.x; c < channels; c += blockDim.x)
            out[t * out_stride + c] =
                z < 0 ? static_cast<T>(0.0f) : static_cast<T>(scale * static_cast<float>(table[z * table_stride + c]));
    }
}

// One workgroup per type and 256 channels: it goes over the atoms' types and
// adds the rows of its own, in their order.
template <class T, class I>
__global__ void __launch_bounds__(256) k_embed_gradient(const I* __restrict__ types, i64 tokens,
                                                        const T* __restrict__ grad, i64 grad_stride, i64 num_types,
                                                        i64 channels, float scale, T* __restrict__ out,
                                                        i64 out_stride) {
    __shared__ unsigned long long mine[4];
    const int v = static_cast<int>(blockIdx.x);
    const i64 c = static_cast<i64>(blockIdx.y) * 256 + threadIdx.x;
    float sum = 0.0f;
    for (i64 t0 = 0; t0 < tokens; t0 += 256) {
        const i64 t = t0 + threadIdx.x;
        const unsigned long long m = __ballot(t < tokens && type_of(types, t, num_types) == v);
        if (threadIdx.x % 64 == 0) mine[threadIdx.x / 64] = m;
        __syncthreads();
        for (int w = 0; w < 4; ++w)
            for (unsigned long long left = mine[w]; left; left &= left - 1) {
                const i64 row = t0 + 64 * w + __builtin_ctzll(left);
                if (c < channels) sum += static_cast<float>(grad[row * grad_stride + c]);
            }
        __syncthreads();
    }
    if (c < channels) out[v * out_stride + c] = static_cast<T>(scale * sum);
}

template <class F>
void with_index(int32_t wide, F&& f) {
    if (wide)
        f(std::int64_t{});
    else
        f(std::int32_t{});
}

void check_embed(const void* types, i64 tokens, i64 num_types, i64 channels, int dtype) {
    require(tokens >= 0 && tokens < (1LL << 31), "tokens must be in [0, 2^31)");
    require(num_types >= 0 && num_types < (1LL << 31), "num_types must be in [0, 2^31)");
    require(channels >= 0 && channels < (1LL << 31), "channels must be in [0, 2^31)");
    require(dtype >= SMX_DTYPE_F32 && dtype <= SMX_DTYPE_F16, "unknown dtype code");
    require(tokens == 0 || types, "types is NULL");
}

}  // namespace
}  // namespace node
}  // namespace smx

using namespace smx;
using namespace smx::node;

extern "C" {

int32_t smx_embed(const void* types, int32_t types_are_64bit, int64_t tokens, const void* table, int64_t table_stride,
                  int64_t num_types, int64_t channels, int32_t dtype, float scale, void* out, int64_t out_stride,
                  void* stream) {
    return guarded([&] {
        check_embed(types, tokens, num_types, channels, dtype);
        check_rows(table, table_stride, num_types, channels, dtype, "table");
        check_rows(out, out_stride, tokens, channels, dtype, "out");
        if (tokens == 0 || channels == 0) return;
        with_dtype(dtype, [&](auto t) {
            using T = decltype(t);
            with_index(types_are_64bit, [&](auto i) {
                using I = decltype(i);
                k_embed<T, I><<<static_cast<unsigned>(tokens < 65536 ? tokens : 65536), 256, 0,
                                static_cast<hipStream_t>(stream)>>>(
                    static_cast<const I*>(types), tokens, static_cast<const T*>(table), table_stride, num_types,
                    channels, scale, static_cast<T*>(out), out_stride);
                SMX_LAUNCH_CHECK("k_embed");
            });
        });
    });
}

int64_t smx_embed_gradient_workspace(int64_t, int64_t, int64_t) { return 0; }

int32_t smx_embed_gradient(const void* types, int32_t types_are_64bit, int64_t tokens, const void* grad,
                           int64_t grad_stride, int64_t num_types, int64_t channels, int32_t dtype, float scale,
                           void* out, int64_t out_stride, void* workspace, int64_t workspace_bytes, void* stream) {
    return guarded([&] {
        check_embed(types, tokens, num_types, channels, dtype);
        check_rows(grad, grad_stride, tokens, channels, dtype, "grad");
        check_rows(out, out_stride, num_types, channels, dtype, "out");
        check_workspace(workspace, workspace_bytes, smx_embed_gradient_workspace(tokens, num_types, channels));
        if (num_types == 0 || channels == 0) return;
        with_dtype(dtype, [&](auto t) {
            using T = decltype(t);
            with_index(types_are_64bit, [&](auto i) {
                using I = decltype(i);
                k_embed_gradient<T, I>
                    <<<dim3(static_cast<unsigned>(num_types), blocks_for(channels, 256)), 256, 0,
                       static_cast<hipStream_t>(stream)>>>(static_cast<const I*>(types), tokens,
                                                           static_cast<const T*>(grad), grad_stride, num_types,
                                                           channels, scale, static_cast<T*>(out), out_stride);
                SMX_LAUNCH_CHECK("k_embed_gradient");
            });
        });
    });
}

}  // extern "C"
