// The norms before and after a block, fused with its gate and residual scale,
// and their gradients.
//
// With r1 = 1 / sqrt(mean(d^2) + eps), u = d r1, s = sigmoid(g), n = post u:
//   y = x + a s n,   r2 = 1 / sqrt(mean(y^2) + eps), v = y r2,   h = next v
// and backward, from G = dL/dy (as an output) and H = dL/dh:
//   q  = H next,     dx = G + r2 (q - v mean(q v)),              dnext  = sum H v
//   dg = dx a n s (1 - s),   da = sum dx s n,   p = dx a s,      dpost  = sum p u
//   t  = p post,     dd = r1 (t - u mean(t u))
#include "node_ops.hpp"

namespace smx {
namespace node {
namespace {

// Device form of SmxResidualNormArgs and SmxResidualNormGradientArgs.
template <class T>
struct Norm {
    i64 rows;
    int channels;
    int gate_kind;
    float eps;
    const T *x, *d, *gate;
    i64 x_stride, d_stride, gate_stride;
    const float *post, *scale, *next;
    T *y, *h;
    i64 y_stride, h_stride;
    std::uint8_t *h8, *h_scales;
    const T *gy, *gh;
    i64 gy_stride, gh_stride;
    T *dx, *dd, *dgate;
    i64 dx_stride, dd_stride, dgate_stride;
    float *dgate_channel, *dpost, *dscale, *dnext;
};

__device__ __forceinline__ float sigmoid(float g) { return 1.0f / (1.0f + __expf(-g)); }

template <class T>
__device__ __forceinline__ float gate_of(const Norm<T>& a, i64 r, int c) {
    switch (a.gate_kind) {
        case SMX_GATE_FULL: return sigmoid(static_cast<float>(a.gate[r * a.gate_stride + c]));
        case SMX_GATE_CHANNEL: return sigmoid(static_cast<float>(a.gate[c]));
        case SMX_GATE_ROW: return sigmoid(static_cast<float>(a.gate[r * a.gate_stride]));
        default: return 1.0f;
    }
}

template <class T>
__device__ __forceinline__ float y_of(const Norm<T>& a, i64 r, int c, float r1) {
    const float x = static_cast<float>(a.x[r * a.x_stride + c]);
    if (!a.d) return x;
    const float n = a.post[c] * static_cast<float>(a.d[r * a.d_stride + c]) * r1;
    return x + (a.scale ? a.scale[c] : 1.0f) * gate_of(a, r, c) * n;
}

// Sum over a workgroup of 256 threads; every thread gets it.
__device__ __forceinline__ float group_sum(float v, float* room) {
    v = wave_total<64>(v);
    __syncthreads();
    if (threadIdx.x % 64 == 0) room[threadIdx.x / 64] = v;
    __syncthreads();
    return (room[0] + room[1]) + (room[2] + room[3]);
}

template <class T>
__device__ __forceinline__ float d_norm(const Norm<T>& a, i64 r, float* room) {
    if (!a.d) return 0.0f;
    float s = 0.0f;
    for (int c = threadIdx.x; c < a.channels; c += 256) {
        const float d = static_cast<float>(a.d[r * a.d_stride + c]);
        s += d * d;
    }
    return 1.0f / sqrtf(group_sum(s, room) / static_cast<float>(a.channels) + a.eps);
}

template <class T>
__device__ __forceinline__ float y_norm(const Norm<T>& a, i64 r, float r1, float* room) {
    float s = 0.0f;
    for (int c = threadIdx.x; c < a.channels; c += 256) {
        const float y = y_of(a, r, c, r1);
        s += y * y;
    }
    return 1.0f / sqrtf(group_sum(s, room) / static_cast<float>(a.channels) + a.eps);
}

// One workgroup per row, reading the row again for each of its sums.
template <class T>
__global__ void __launch_bounds__(256) k_residual_norm(Norm<T> a) {
    __shared__ float room[4], blocks[4];
    for (i64 r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const float r1 = d_norm(a, r, room);
        const float r2 = a.next ? y_norm(a, r, r1, room) : 0.0f;
        const int padded = a.h8 ? (a.channels + 255) / 256 * 256 : a.channels;
        for (int c0 = 0; c0 < padded; c0 += 256) {
            const int c = c0 + threadIdx.x;
            const bool in = c < a.channels;
            const float y = in ? y_of(a, r, c, r1) : 0.0f;
            const float h = in && a.next ? a.next[c] * y * r2 : 0.0f;
            if (a.h8) {
                float top = finite_magnitude(h);
                for (int o = 32; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
                __syncthreads();
                if (threadIdx.x % 64 == 0) blocks[threadIdx.x / 64] = top;
                __syncthreads();
                const int w = threadIdx.x / 128 * 2;
                const int byte = block_scale_byte(fmaxf(blocks[w], blocks[w + 1]));
                const int width = (a.channels + 127) / 128 * 128;
                if (c < width) {
                    a.h8[r * width + c] = static_cast<std::uint8_t>(
                        e4m3_four(h, 0.0f, 0.0f, 0.0f, block_inverse_scale(byte)) & 0xff);
                    const int pitch = (width / 128 + 3) / 4 * 4;
                    if (c % 128 == 0) a.h_scales[r * pitch + c / 128] = static_cast<std::uint8_t>(byte);
                    if (c == 0)
                        for (int b = width / 128; b < pitch; ++b) a.h_scales[r * pitch + b] = 0;
                }
            } else if (in && a.next) {
                a.h[r * a.h_stride + c] = static_cast<T>(h);
            }
            if (in && a.y) a.y[r * a.y_stride + c] = static_cast<T>(y);
        }
    }
}

// One workgroup per row: its outputs, and the row's r1, r2 and mean(q v) for
// the sums over rows.
template <class T>
__global__ void __launch_bounds__(256) k_norm_gradient_rows(Norm<T> a, float* __restrict__ stats) {
    __shared__ float room[4];
    const float inv = 1.0f / static_cast<float>(a.channels);
    for (i64 r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const float r1 = d_norm(a, r, room);
        float r2 = 0.0f, m2 = 0.0f;
        if (a.gh) {
            r2 = y_norm(a, r, r1, room);
            float s = 0.0f;
            for (int c = threadIdx.x; c < a.channels; c += 256)
                s += static_cast<float>(a.gh[r * a.gh_stride + c]) * a.next[c] * y_of(a, r, c, r1) * r2;
            m2 = group_sum(s, room) * inv;
        }
        const auto dx_of = [&](int c) {
            float g = a.gy ? static_cast<float>(a.gy[r * a.gy_stride + c]) : 0.0f;
            if (a.gh)
                g += r2 * (static_cast<float>(a.gh[r * a.gh_stride + c]) * a.next[c] - y_of(a, r, c, r1) * r2 * m2);
            return g;
        };
        float m1 = 0.0f, row_gate = 0.0f;
        if (a.d) {
            float s = 0.0f, k = 0.0f;
            for (int c = threadIdx.x; c < a.channels; c += 256) {
                const float dx = dx_of(c), u = static_cast<float>(a.d[r * a.d_stride + c]) * r1;
                const float sc = a.scale ? a.scale[c] : 1.0f, sg = gate_of(a, r, c);
                s += dx * sc * sg * a.post[c] * u;
                k += dx * sc * a.post[c] * u * sg * (1.0f - sg);
            }
            m1 = group_sum(s, room) * inv;
            row_gate = group_sum(k, room);
        }
        __syncthreads();  // dx may lie where gy does
        for (int c = threadIdx.x; c < a.channels; c += 256) {
            const float dx = dx_of(c);
            if (a.d) {
                const float u = static_cast<float>(a.d[r * a.d_stride + c]) * r1;
                const float sc = a.scale ? a.scale[c] : 1.0f, sg = gate_of(a, r, c);
                if (a.dd) a.dd[r * a.dd_stride + c] = static_cast<T>(r1 * (dx * sc * sg * a.post[c] - u * m1));
                if (a.dgate && a.gate_kind == SMX_GATE_FULL)
                    a.dgate[r * a.dgate_stride + c] = static_cast<T>(dx * sc * a.post[c] * u * sg * (1.0f - sg));
            }
            if (a.dx) a.dx[r * a.dx_stride + c] = static_cast<T>(dx);
        }
        if (threadIdx.x == 0) {
            if (a.dgate && a.gate_kind == SMX_GATE_ROW) a.dgate[r * a.dgate_stride] = static_cast<T>(row_gate);
            stats[3 * r] = r1;
            stats[3 * r + 1] = r2;
            stats[3 * r + 2] = m2;
        }
    }
}

// The sums over rows: 64 channels a workgroup, sixteen of its waves' rows at a time.
template <class T>
__global__ void __launch_bounds__(1024) k_norm_gradient_channels(Norm<T> a, const float* __restrict__ stats) {
    __shared__ float part[16][4][64];
    const int lane = threadIdx.x % 64, wave = threadIdx.x / 64, c = blockIdx.x * 64 + lane;
    float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if (c < a.channels)
        for (i64 r = wave; r < a.rows; r += 16) {
            const float r1 = stats[3 * r], r2 = stats[3 * r + 1], m2 = stats[3 * r + 2];
            float dx = a.gy ? static_cast<float>(a.gy[r * a.gy_stride + c]) : 0.0f;
            if (a.gh) {
                const float gh = static_cast<float>(a.gh[r * a.gh_stride + c]), v = y_of(a, r, c, r1) * r2;
                dx += r2 * (gh * a.next[c] - v * m2);
                s[3] += gh * v;
            }
            if (a.d) {
                const float u = static_cast<float>(a.d[r * a.d_stride + c]) * r1;
                const float sc = a.scale ? a.scale[c] : 1.0f, sg = gate_of(a, r, c);
                s[0] += dx * sc * a.post[c] * u * sg * (1.0f - sg);
                s[1] += dx * sc * sg * u;
                s[2] += dx * sg * a.post[c] * u;
            }
        }
    for (int k = 0; k < 4; ++k) part[wave][k][lane] = s[k];
    __syncthreads();
    if (wave >= 4 || c >= a.channels) return;
    float* const out = wave == 0 ? (a.gate_kind == SMX_GATE_CHANNEL ? a.dgate_channel : nullptr)
                                 : wave == 1 ? a.dpost : wave == 2 ? a.dscale : a.dnext;
    if (!out) return;
    float sum = 0.0f;
    for (int w = 0; w < 16; ++w) sum += part[w][wave][lane];
    out[c] = sum;
}

void check_norm(const SmxResidualNormArgs& a) {
    require(a.rows >= 0 && a.rows < (1LL << 31), "rows must be in [0, 2^31)");
    require(a.channels >= 1, "channels must be at least 1");
    if (a.channels > 16384) throw std::domain_error("the residual norm has no kernel for more than 16384 channels");
    require(a.dtype >= SMX_DTYPE_F32 && a.dtype <= SMX_DTYPE_F16, "unknown dtype code");
    require(a.eps >= 0.0f, "eps must not be negative");
    check_rows(a.x, a.x_stride, a.rows, a.channels, a.dtype, "x");
    if (a.d) {
        check_rows(a.d, a.d_stride, a.rows, a.channels, a.dtype, "d");
        require(a.post, "post is NULL");
        require(a.gate_kind >= SMX_GATE_NONE && a.gate_kind <= SMX_GATE_ROW, "unknown gate kind");
        if (a.gate_kind == SMX_GATE_FULL) check_rows(a.gate, a.gate_stride, a.rows, a.channels, a.dtype, "gate");
        if (a.gate_kind == SMX_GATE_CHANNEL) check_rows(a.gate, a.channels, 1, a.channels, a.dtype, "gate");
        if (a.gate_kind == SMX_GATE_ROW) check_rows(a.gate, a.gate_stride, a.rows, 1, a.dtype, "gate");
    }
    for (const float* p : {a.post, a.scale, a.next}) require(aligned(p, 4), "post, scale and next must be aligned to their values");
}

template <class T>
Norm<T> device_args(const SmxResidualNormArgs& a) {
    Norm<T> n{};
    n.rows = a.rows;
    n.channels = static_cast<int>(a.channels);
    n.gate_kind = a.d || a.rows == 0 ? a.gate_kind : SMX_GATE_NONE;
    n.eps = a.eps;
    n.x = static_cast<const T*>(a.x);
    n.d = static_cast<const T*>(a.d);
    n.gate = static_cast<const T*>(a.gate);
    n.x_stride = a.x_stride;
    n.d_stride = a.d_stride;
    n.gate_stride = a.gate_stride;
    n.post = a.post;
    n.scale = a.scale;
    n.next = a.next;
    return n;
}

}  // namespace
}  // namespace node
}  // namespace smx

using namespace smx;
using namespace smx::node;

extern "C" {

int32_t smx_residual_norm(const SmxResidualNormArgs* args, void* stream) {
    return guarded([&] {
        require(args && args->struct_size == sizeof(SmxResidualNormArgs), "args is NULL or has another struct_size");
        const SmxResidualNormArgs& a = *args;
        check_norm(a);
        if (a.y) check_rows(a.y, a.y_stride, a.rows, a.channels, a.dtype, "y");
        require(!a.h || a.next, "h is asked for without next");
        require(!a.next || a.h || a.rows == 0, "h is NULL");
        require(!a.h_scales || a.h, "h_scales without h");
        require(!a.h_scales || (aligned(a.h, 16) && aligned(a.h_scales, 16)), "8-bit blocks must be 16-byte aligned");
        if (a.h && !a.h_scales) check_rows(a.h, a.h_stride, a.rows, a.channels, a.dtype, "h");
        require(a.y || a.h || a.rows == 0, "neither y nor h is asked for");
        if (a.rows == 0) return;
        with_dtype(a.dtype, [&](auto t) {
            using T = decltype(t);
            Norm<T> n = device_args<T>(a);
            n.y = static_cast<T*>(a.y);
            n.y_stride = a.y_stride;
            if (a.h_scales) {
                n.h8 = static_cast<std::uint8_t*>(a.h);
                n.h_scales = a.h_scales;
            } else {
                n.h = static_cast<T*>(a.h);
                n.h_stride = a.h_stride;
            }
            k_residual_norm<T><<<static_cast<unsigned>(a.rows < 65536 ? a.rows : 65536), 256, 0,
                                 static_cast<hipStream_t>(stream)>>>(n);
            SMX_LAUNCH_CHECK("k_residual_norm");
        });
    });
}

int64_t smx_residual_norm_gradient_workspace(int64_t rows, int64_t) { return rows > 0 ? 12 * rows : 0; }

int32_t smx_residual_norm_gradient(const SmxResidualNormGradientArgs* args, void* stream) {
    return guarded([&] {
        require(args && args->forward.struct_size == sizeof(SmxResidualNormArgs),
                "args is NULL or has another struct_size");
        const SmxResidualNormGradientArgs& g = *args;
        const SmxResidualNormArgs& a = g.forward;
        check_norm(a);
        require(!g.grad_h || a.next, "grad_h without next");
        if (g.grad_y) check_rows(g.grad_y, g.grad_y_stride, a.rows, a.channels, a.dtype, "grad_y");
        if (g.grad_h) check_rows(g.grad_h, g.grad_h_stride, a.rows, a.channels, a.dtype, "grad_h");
        if (g.dx) check_rows(g.dx, g.dx_stride, a.rows, a.channels, a.dtype, "dx");
        require(a.d || a.rows == 0 || (!g.dd && !g.dgate && !g.dpost && !g.dscale), "gradients of d, gate, post or scale without d");
        require(!g.dgate || a.gate_kind != SMX_GATE_NONE, "dgate without a gate");
        require(!g.dscale || a.scale, "dscale without scale");
        require(!g.dnext || a.next, "dnext without next");
        if (g.dd) check_rows(g.dd, g.dd_stride, a.rows, a.channels, a.dtype, "dd");
        if (g.dgate && a.gate_kind == SMX_GATE_FULL)
            check_rows(g.dgate, g.dgate_stride, a.rows, a.channels, a.dtype, "dgate");
        if (g.dgate && a.gate_kind == SMX_GATE_ROW) check_rows(g.dgate, g.dgate_stride, a.rows, 1, a.dtype, "dgate");
        if (g.dgate && a.gate_kind == SMX_GATE_CHANNEL) require(aligned(g.dgate, 4), "dgate is not aligned to its values");
        check_workspace(g.workspace, g.workspace_bytes, smx_residual_norm_gradient_workspace(a.rows, a.channels));
        with_dtype(a.dtype, [&](auto t) {
            using T = decltype(t);
            Norm<T> n = device_args<T>(a);
            n.gy = static_cast<const T*>(g.grad_y);
            n.gh = static_cast<const T*>(g.grad_h);
            n.gy_stride = g.grad_y_stride;
            n.gh_stride = g.grad_h_stride;
            n.dx = static_cast<T*>(g.dx);
            n.dd = static_cast<T*>(g.dd);
            n.dx_stride = g.dx_stride;
            n.dd_stride = g.dd_stride;
            if (a.gate_kind == SMX_GATE_CHANNEL)
                n.dgate_channel = static_cast<float*>(g.dgate);
            else
                n.dgate = static_cast<T*>(g.dgate);
            n.dgate_stride = g.dgate_stride;
            n.dpost = g.dpost;
            n.dscale = g.dscale;
            n.dnext = g.dnext;
            float* const stats = static_cast<float*>(g.workspace);
            if (a.rows > 0) {
                k_norm_gradient_rows<T><<<static_cast<unsigned>(a.rows < 65536 ? a.rows : 65536), 256, 0,
                                          static_cast<hipStream_t>(stream)>>>(n, stats);
                SMX_LAUNCH_CHECK("k_norm_gradient_rows");
            }
            if (n.dgate_channel || n.dpost || n.dscale || n.dnext) {
                k_norm_gradient_channels<T><<<blocks_for(a.channels, 64), 1024, 0, static_cast<hipStream_t>(stream)>>>(
                    n, stats);
                SMX_LAUNCH_CHECK("k_norm_gradient_channels");
            }
        });
    });
}

}  // extern "C"
