// The norms before and after a block, fused with its gate and residual scale,
// and their gradients.
//
// With r1 = 1 / sqrt(mean(d^2) + eps), u = d r1, s = sigmoid(g), n = post u:
//   y = x + a s n,   r2 = 1 / sqrt(mean(y^2) + eps), v = y r2,   h = next v
// and backward, from G = dL/dy (as an output) and H = dL/dh:
//   q  = H next,     dx = G + r2 (q - v mean(q v)),              dnext  = sum H v
//   dg = dx a n s (1 - s),   da = sum dx s n,   p = dx a s,      dpost  = sum p u
//   t  = p post,     dd = r1 (t - u mean(t u))
#include <variant>

#include "node_ops.hpp"

#include "group_sum.hpp"

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
    T* dgate_channel;
    float *dpost, *dscale, *dnext;
};

// e^-a for a >= 0 (an infinity gives 0).  The hardware exponential of a log2(e), whose rounding alone is a 2^-24 of the
// result: 16-bit rows take it as it is (at a logit of 80, 2^-18).  For FP32 rows what the rounding left out, and what log2(e)
// has beyond FP32, is added to first order: 2^-22 for every a.
template <class T>
__device__ __forceinline__ float exp_minus(float a) {
    const float hi = a * -1.44269504f, e = __builtin_amdgcn_exp2f(hi);
    if constexpr (sizeof(T) == 4) {
        const float lo = __builtin_fmaf(a, -1.92596303e-8f, __builtin_fmaf(a, -1.44269504f, -hi));
        return a < 128.0f ? __builtin_fmaf(e * 0.693147181f, lo, e) : e;
    }
    return e;
}

// s = 1 / (1 + e^-g), and 1 - s as a quotient of its own: as a difference it has no digit left from g = 17 on.
struct Gate {
    float s, rest;
};

template <class T>
__device__ __forceinline__ Gate gate_of(float g) {
    const float t = exp_minus<T>(__builtin_fabsf(g)), near = __builtin_amdgcn_rcpf(1.0f + t), far = t * near;
    return g < 0.0f ? Gate{far, near} : Gate{near, far};
}

// Threads of a workgroup with G lanes a row: several rows' lanes up to a wave each, one row's above
// (whose sums wait at barriers, so no other row may share the workgroup).
constexpr int threads_of(int g) { return g > 64 ? g : 256; }

// What a lane keeps of the channels it holds, for all its rows: scale * post (times the gate, where
// it is the channel's) and next.
template <class T>
__device__ __forceinline__ void load_channels(const Norm<T>& a, int c, float (&step)[8], float (&next)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) step[i] = next[i] = 0.0f;
    if (a.d) {
        float v[8];
        load_eight(a.post, c, a.channels, step);
        if (a.scale) {
            load_eight(a.scale, c, a.channels, v);
#pragma unroll
            for (int i = 0; i < 8; ++i) step[i] *= v[i];
        }
        if (a.gate_kind == SMX_GATE_CHANNEL) {
            load_eight(a.gate, c, a.channels, v);
#pragma unroll
            for (int i = 0; i < 8; ++i) step[i] *= gate_of<T>(v[i]).s;
        }
    }
    if (a.next) load_eight(a.next, c, a.channels, next);
}

// A lane's share of a row as it lies in memory; FULL: a gate for each value, which takes registers that the other
// kernels do without (8192 x 8192 FP32 gradient without it: 424 -> 314 us).
template <class T, bool FULL>
struct Share {
    Eight<T> x, d;
    std::conditional_t<FULL, Eight<T>, std::monostate> g;
};

template <class T, bool FULL>
__device__ __forceinline__ void load_share(const Norm<T>& a, i64 r, int c, Share<T, FULL>& s) {
    s.x = load_pack(a.x + r * a.x_stride, c, a.channels);
    if (!a.d) return;
    s.d = load_pack(a.d + r * a.d_stride, c, a.channels);
    if constexpr (FULL) s.g = load_pack(a.gate + r * a.gate_stride, c, a.channels);
}

template <class T, bool FULL>
__device__ __forceinline__ void settle_share(const Norm<T>& a, int c, Share<T, FULL>& s) {
    settle(s.x, c, a.channels);
    if (!a.d) return;
    settle(s.d, c, a.channels);
    if constexpr (FULL) settle(s.g, c, a.channels);
}

template <class T>
__device__ __forceinline__ T row_gate_of(const Norm<T>& a, i64 r) {
    return a.gate_kind == SMX_GATE_ROW ? a.gate[r * a.gate_stride] : static_cast<T>(0.0f);
}

// The gate of channel i of a lane's eight, where it is not in the channel's step.
template <class T, bool FULL>
__device__ __forceinline__ Gate gate_at(const Share<T, FULL>& s, int i, const Gate& row_gate) {
    if constexpr (FULL)
        return gate_of<T>(s.g[i]);
    else
        return row_gate;
}

template <class T>
__device__ __forceinline__ float square_sum(const Eight<T>& d) {
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) s += d[i] * d[i];
    return s;
}

// G lanes a row, each N times eight neighbouring values in registers, so that
// a row is read once and its two sums stay between lanes; a lane keeps its channels'
// weights for all its rows.  A group of 128 channels is 16 lanes, which is where an 8-bit block's
// scale is found.  Bound by memory: five values of 16 bits a channel at 5.0 TB/s (32768 x 2048, 133 us) to 5.9 (60000 x 256,
// 26 us); rows that end within eight channels lose a tenth (6791 x 999 FP32 24.9 us, x 1000 22.7).
template <class T, bool FULL, int G, int N>
__global__ void __launch_bounds__(threads_of(G)) k_residual_norm(Norm<T> a) {
    constexpr int kThreads = threads_of(G), kGroups = kThreads / G;
    __shared__ typename GroupSum<G, 1>::Room room;
    const int lane = threadIdx.x % G;
    const float inv = 1.0f / static_cast<float>(a.channels);
    float step[N][8], next[N][8];
#pragma unroll
    for (int n = 0; n < N; ++n) load_channels(a, 8 * (lane + G * n), step[n], next[n]);
    int turn = 0;
    for (i64 r = static_cast<i64>(blockIdx.x) * kGroups + threadIdx.x / G; r < a.rows;
         r += static_cast<i64>(gridDim.x) * kGroups) {
        Share<T, FULL> s[N];
        float sum[1] = {0.0f};
#pragma unroll
        for (int n = 0; n < N; ++n) load_share(a, r, 8 * (lane + G * n), s[n]);
#pragma unroll
        for (int n = 0; n < N; ++n) {
            settle_share(a, 8 * (lane + G * n), s[n]);
            if (a.d) sum[0] += square_sum(s[n].d);
        }
        float r1 = 0.0f;
        Gate row_gate{1.0f, 0.0f};
        if (a.d) {
            if (a.gate_kind == SMX_GATE_ROW) row_gate = gate_of<T>(static_cast<float>(row_gate_of(a, r)));
            GroupSum<G, 1>::sum(sum, room, turn);
            r1 = rsqrtf(sum[0] * inv + a.eps);
        }
        float y[N][8];
        sum[0] = 0.0f;
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const int c = 8 * (lane + G * n);
#pragma unroll
            for (int i = 0; i < 8; ++i) y[n][i] = s[n].x[i];
            if (a.d) {
#pragma unroll
                for (int i = 0; i < 8; ++i) y[n][i] += step[n][i] * gate_at(s[n], i, row_gate).s * (s[n].d[i] * r1);
            }
            if (a.y) store_eight(a.y + r * a.y_stride, c, a.channels, y[n]);
#pragma unroll
            for (int i = 0; i < 8; ++i) sum[0] += c + i < a.channels ? y[n][i] * y[n][i] : 0.0f;
        }
        if (!a.next) continue;
        GroupSum<G, 1>::sum(sum, room, turn);
        const float r2 = rsqrtf(sum[0] * inv + a.eps);
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const int c = 8 * (lane + G * n);
#pragma unroll
            for (int i = 0; i < 8; ++i) y[n][i] = c + i < a.channels ? next[n][i] * (y[n][i] * r2) : 0.0f;
            if (a.h8) {
                const int pitch = (a.channels + kBlock - 1) / kBlock * kBlock, blocks = pitch / kBlock;
                const int scale_pitch = (blocks + 3) / 4 * 4, k = c / kBlock;
                const int byte = block_scale_byte(row_max(top_of(y[n])));
                if (c < pitch) {
                    *reinterpret_cast<uint2*>(a.h8 + r * pitch + c) = e4m3_eight(y[n], block_inverse_scale(byte));
                    std::uint8_t* const at = a.h_scales + r * scale_pitch + k;
                    const int sub = lane % 16;
                    if (sub == 0) *at = static_cast<std::uint8_t>(byte);
                    if (k + 1 == blocks && sub > 0 && k + sub < scale_pitch) at[sub] = 0;
                }
            } else {
                store_eight(a.h + r * a.h_stride, c, a.channels, y[n]);
            }
        }
    }
}

// What a workgroup adds up over its rows: S = sum dx s u and dnext.  Where the gate is the
// channel's, or there is none, every other gradient of a channel vector is S times
// constants of the channel, and dpost = a S, dscale = post S always.
constexpr int kSums = 2;

// The gradient of a row in one reading of it, as above, in two rounds of sums: mean(d^2), and then,
// with f = a post s and dx = G + r2 q - r2^2 m y, m = r2 mean(q y), those of y^2, q y and the three parts of
//   sum t u = sum G f u + r2 sum q f u - r2^2 m sum y f u,
// which is also a row gate's gradient over 1 - s.  The next row is read while
// one is worked on (6791 x 999 FP32: 47.5 us, 54.9 without; 43.8 since rows' ends are loaded like the rest).  Bound by memory
// with two or three waves a SIMD: eight values a channel at 4.7 TB/s (32768 x 2048 bf16, 228 us; 8192 x 8192 FP32 443 us at
// 4.8); above 8,192 channels a lane has sixteen values of each array in 128 registers and spills (4000 x 16384 bf16: 684 us,
// 1.5 TB/s).  The sums over rows stay in registers over all rows of a group, are joined in LDS for the workgroup's groups, and
// leave as one part [kSums][channels] a workgroup.
template <class T, bool FULL, int G, int N>
__global__ void __launch_bounds__(threads_of(G)) k_norm_gradient(Norm<T> a, float* __restrict__ parts) {
    constexpr int kThreads = threads_of(G), kGroups = kThreads / G;
    __shared__ union {
        typename GradientSums<G>::Room room;
        float join[kGroups > 1 ? kGroups : 1][kGroups > 1 ? G * 8 * N : 1];
    } lds;
    struct Row {
        Share<T, FULL> s[N];
        Eight<T> gy[N], gh[N];
        T gate;
    };
    const int lane = threadIdx.x % G;
    const float inv = 1.0f / static_cast<float>(a.channels);
    float step[N][8], next[N][8], acc[kSums][N][8];
#pragma unroll
    for (int n = 0; n < N; ++n) {
        load_channels(a, 8 * (lane + G * n), step[n], next[n]);
#pragma unroll
        for (int k = 0; k < kSums; ++k)
#pragma unroll
            for (int i = 0; i < 8; ++i) acc[k][n][i] = 0.0f;
    }
    const auto read = [&](i64 r, Row& row) {
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const int c = 8 * (lane + G * n);
            load_share(a, r, c, row.s[n]);
            if (a.gy) row.gy[n] = load_pack(a.gy + r * a.gy_stride, c, a.channels);
            if (a.gh) row.gh[n] = load_pack(a.gh + r * a.gh_stride, c, a.channels);
        }
        row.gate = row_gate_of(a, r);
    };
    // (a workgroup of 16 waves has half the registers a lane: other waves' work covers its reading)
    constexpr bool kAhead = threads_of(G) <= 512;
    const i64 hop = static_cast<i64>(gridDim.x) * kGroups;
    GradientSums<G> sums{lds.room};
    i64 r = static_cast<i64>(blockIdx.x) * kGroups + threadIdx.x / G;
    Row row, ahead;
    if (kAhead && r < a.rows) read(r, row);
    for (; r < a.rows; r += hop) {
        if constexpr (!kAhead)
            read(r, row);
        else if (r + hop < a.rows)
            read(r + hop, ahead);
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const int c = 8 * (lane + G * n);
            settle_share(a, c, row.s[n]);
            if (a.gy) settle(row.gy[n], c, a.channels);
            if (a.gh) settle(row.gh[n], c, a.channels);
        }
        float r1 = 0.0f;
        const Gate row_gate = a.gate_kind == SMX_GATE_ROW ? gate_of<T>(static_cast<float>(row.gate)) : Gate{1.0f, 0.0f};
        if (a.d) {
            float sum[1] = {0.0f};
#pragma unroll
            for (int n = 0; n < N; ++n) sum[0] += square_sum(row.s[n].d);
            sums.sum(sum);
            r1 = rsqrtf(sum[0] * inv + a.eps);
        }
        float y[N][8], sum[5] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
        Gate kept[N][8];  // (where a lane has the registers; else the gates are formed again in the second round)
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const int c = 8 * (lane + G * n);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                y[n][i] = row.s[n].x[i];
                const float q = a.gh ? row.gh[n][i] * next[n][i] : 0.0f;
                if (a.d) {
                    kept[n][i] = gate_at(row.s[n], i, row_gate);
                    const float fu = step[n][i] * kept[n][i].s * (row.s[n].d[i] * r1);
                    y[n][i] += fu;
                    sum[2] += a.gy ? row.gy[n][i] * fu : 0.0f;
                    sum[3] += q * fu;
                    sum[4] += y[n][i] * fu;
                }
                sum[0] += c + i < a.channels ? y[n][i] * y[n][i] : 0.0f;
                sum[1] += q * y[n][i];
            }
        }
        sums.sum(sum);
        const float r2 = a.gh ? rsqrtf(sum[0] * inv + a.eps) : 0.0f;
        if constexpr (!kAhead) {
            // work gate and step out again below: sixteen registers less over the sums' barrier
#pragma unroll
            for (int n = 0; n < N; ++n)
#pragma unroll
                for (int i = 0; i < Eight<T>::kWords; ++i) {
                    if constexpr (FULL) asm volatile("" : "+v"(row.s[n].g.w[i]));
                    asm volatile("" : "+v"(row.s[n].d.w[i]));
                    asm volatile("" : "+v"(row.gh[n].w[i]));
                }
        }
        // (without h's gradient, sums that take y are not looked at: they may be infinite)
        const float ry = a.gh ? r2 * r2 * (r2 * (sum[1] * inv)) : 0.0f;
        const float tu = a.gh ? sum[2] + r2 * sum[3] - ry * sum[4] : sum[2], m1 = tu * inv;
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const int c = 8 * (lane + G * n);
            float dx[8], dd[8], dg[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                dx[i] = a.gy ? row.gy[n][i] : 0.0f;
                if (a.gh) {
                    const float g = row.gh[n][i];
                    dx[i] += r2 * (g * next[n][i]) - ry * y[n][i];
                    acc[1][n][i] += g * (y[n][i] * r2);
                }
                if (a.d) {
                    const Gate gate = kAhead ? kept[n][i] : gate_at(row.s[n], i, row_gate);
                    const float u = row.s[n].d[i] * r1, t = dx[i] * (step[n][i] * gate.s);
                    acc[0][n][i] += dx[i] * (gate.s * u);
                    dd[i] = r1 * (t - u * m1);
                    dg[i] = t * u * gate.rest;
                }
            }
            if (a.dx) store_eight(a.dx + r * a.dx_stride, c, a.channels, dx);
            if (a.dd) store_eight(a.dd + r * a.dd_stride, c, a.channels, dd);
            if (FULL && a.dgate) store_eight(a.dgate + r * a.dgate_stride, c, a.channels, dg);
        }
        if (a.dgate && a.gate_kind == SMX_GATE_ROW && lane == 0)
            a.dgate[r * a.dgate_stride] = static_cast<T>(tu * row_gate.rest);
        if constexpr (kAhead) row = ahead;
    }
    if (!parts) return;
    float* const part = parts + static_cast<i64>(blockIdx.x) * kSums * a.channels;
#pragma unroll
    for (int k = 0; k < kSums; ++k) {
        if constexpr (kGroups > 1) {
            __syncthreads();
#pragma unroll
            for (int n = 0; n < N; ++n)
#pragma unroll
                for (int i = 0; i < 8; ++i) lds.join[threadIdx.x / G][8 * (lane + G * n) + i] = acc[k][n][i];
            __syncthreads();
            for (int c = threadIdx.x; c < a.channels; c += kThreads) {
                float v = lds.join[0][c];
#pragma unroll
                for (int g = 1; g < kGroups; ++g) v += lds.join[g][c];
                part[k * a.channels + c] = v;
            }
        } else {
#pragma unroll
            for (int n = 0; n < N; ++n) store_eight(part + k * a.channels, 8 * (lane + G * n), a.channels, acc[k][n]);
        }
    }
}

// Adds the workgroups' parts up.
template <class T>
__global__ void __launch_bounds__(1024) k_norm_gradient_join(Norm<T> a, const float* __restrict__ parts, int count) {
    const int c = blockIdx.x * kJoined + threadIdx.x % kJoined, k = blockIdx.y;
    if (k == 0 ? !a.d : !a.dnext) return;
    const float sum = sum_of_parts(parts + static_cast<i64>(k) * a.channels + c, static_cast<i64>(kSums) * a.channels, count,
                                   c < a.channels);
    if (threadIdx.x >= kJoined || c >= a.channels) return;
    if (k == 1) {
        a.dnext[c] = sum;
        return;
    }
    const float scale = a.scale ? a.scale[c] : 1.0f;
    Gate gate{1.0f, 0.0f};
    if (a.gate_kind == SMX_GATE_CHANNEL) {  // S was summed without the channel's gate
        gate = gate_of<T>(static_cast<float>(a.gate[c]));
        if (a.dgate_channel) a.dgate_channel[c] = static_cast<T>(sum * a.post[c] * scale * gate.s * gate.rest);
    }
    if (a.dpost) a.dpost[c] = sum * scale * gate.s;
    if (a.dscale) a.dscale[c] = sum * a.post[c] * gate.s;
}

// The channel vectors' gradients of no rows.
template <class T>
__global__ void __launch_bounds__(256) k_norm_gradient_none(Norm<T> a) {
    const int c = blockIdx.x * 256 + threadIdx.x;
    if (c >= a.channels) return;
    if (a.dgate_channel) a.dgate_channel[c] = static_cast<T>(0.0f);
    for (float* const out : {a.dpost, a.dscale, a.dnext})
        if (out) out[c] = 0.0f;
}

// f(lanes a row, times eight values a lane) for the forward kernel: up to 16 values
// a lane, whose row then is in at most 64 lanes up to 1,024 channels.
template <class F>
void with_forward_shape(int channels, F&& f) {
    using std::integral_constant;
    const auto go = [&](auto g, auto n) { f(g, n); };
#define SMX_SHAPE(MOST, G, N) \
    if (channels <= MOST) return go(integral_constant<int, G>{}, integral_constant<int, N>{});
    SMX_SHAPE(128, 16, 1)
    SMX_SHAPE(256, 32, 1)
    SMX_SHAPE(512, 64, 1)
    SMX_SHAPE(1024, 64, 2)
    SMX_SHAPE(2048, 256, 1)
    SMX_SHAPE(4096, 512, 1)
    SMX_SHAPE(8192, 1024, 1)
    SMX_SHAPE(16384, 1024, 2)
}

// For the gradient, which holds five rows and four sums besides: eight values a lane as far as a
// workgroup goes.
template <class F>
void with_gradient_shape(int channels, F&& f) {
    using std::integral_constant;
    const auto go = [&](auto g, auto n) { f(g, n); };
    SMX_SHAPE(128, 16, 1)
    SMX_SHAPE(256, 32, 1)
    SMX_SHAPE(512, 64, 1)
    SMX_SHAPE(1024, 128, 1)
    SMX_SHAPE(2048, 256, 1)
    SMX_SHAPE(4096, 512, 1)
    SMX_SHAPE(8192, 1024, 1)
    SMX_SHAPE(16384, 1024, 2)
#undef SMX_SHAPE
}

constexpr i64 kUnits = 256;  // compute units

// Workgroups of a gradient call, each of which leaves a part: as many as the card holds at once at two
// waves a SIMD, and at least two rows a group.
i64 gradient_groups(i64 rows, i64 channels) {
    i64 groups = 1, threads = 256;
    with_gradient_shape(static_cast<int>(channels), [&](auto g, auto) {
        threads = threads_of(g.value);
        groups = threads / g.value;
    });
    const i64 full = kUnits * (threads < 512 ? 512 / threads : 1), want = (rows + 2 * groups - 1) / (2 * groups);
    return want < full ? want : full;
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
    n.gate_kind = a.d ? a.gate_kind : SMX_GATE_NONE;
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
            with_forward_shape(n.channels, [&](auto g, auto times) {
                constexpr int G = decltype(g)::value, N = decltype(times)::value;
                constexpr int threads = threads_of(G), groups = threads / G;
                // twice what the card holds: a unit that is done early takes another (300,000 x 100 bf16 76 -> 73 us; four
                // times: 71, but 60,000 x 256 26.3 against 24.8)
                const i64 want = (a.rows + groups - 1) / groups, full = kUnits * (4096 / threads);
                (n.gate_kind == SMX_GATE_FULL ? k_residual_norm<T, true, G, N> : k_residual_norm<T, false, G, N>)<<<
                    static_cast<unsigned>(want < full ? want : full), threads, 0, static_cast<hipStream_t>(stream)>>>(n);
            });
            SMX_LAUNCH_CHECK("k_residual_norm");
        });
    });
}

int64_t smx_residual_norm_gradient_workspace(int64_t rows, int64_t channels) {
    if (rows <= 0 || channels <= 0 || channels > 16384) return 0;
    return 4 * kSums * channels * gradient_groups(rows, channels);
}

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
        require(!g.dgate || (a.gate_kind >= SMX_GATE_FULL && a.gate_kind <= SMX_GATE_ROW), "dgate without a gate");
        require(!g.dscale || a.scale, "dscale without scale");
        require(!g.dnext || a.next, "dnext without next");
        if (g.dd) check_rows(g.dd, g.dd_stride, a.rows, a.channels, a.dtype, "dd");
        if (g.dgate && a.gate_kind == SMX_GATE_FULL)
            check_rows(g.dgate, g.dgate_stride, a.rows, a.channels, a.dtype, "dgate");
        if (g.dgate && a.gate_kind == SMX_GATE_ROW) check_rows(g.dgate, g.dgate_stride, a.rows, 1, a.dtype, "dgate");
        if (g.dgate && a.gate_kind == SMX_GATE_CHANNEL) check_rows(g.dgate, a.channels, 1, a.channels, a.dtype, "dgate");
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
                n.dgate_channel = static_cast<T*>(g.dgate);
            else
                n.dgate = static_cast<T*>(g.dgate);
            n.dgate_stride = g.dgate_stride;
            n.dpost = g.dpost;
            n.dscale = g.dscale;
            n.dnext = g.dnext;
            const bool sums = n.dgate_channel || n.dpost || n.dscale || n.dnext;
            if (a.rows == 0) {
                if (!sums) return;
                k_norm_gradient_none<T><<<blocks_for(a.channels, 256), 256, 0, static_cast<hipStream_t>(stream)>>>(n);
                SMX_LAUNCH_CHECK("k_norm_gradient_none");
                return;
            }
            float* const parts = sums ? static_cast<float*>(g.workspace) : nullptr;
            const i64 count = gradient_groups(a.rows, a.channels);
            with_gradient_shape(n.channels, [&](auto lanes, auto times) {
                constexpr int G = decltype(lanes)::value, N = decltype(times)::value;
                (n.gate_kind == SMX_GATE_FULL ? k_norm_gradient<T, true, G, N> : k_norm_gradient<T, false, G, N>)<<<
                    static_cast<unsigned>(count), threads_of(G), 0, static_cast<hipStream_t>(stream)>>>(n, parts);
            });
            SMX_LAUNCH_CHECK("k_norm_gradient");
            if (sums) {
                k_norm_gradient_join<T><<<dim3(blocks_for(a.channels, kJoined), kSums), 1024, 0,
                                          static_cast<hipStream_t>(stream)>>>(n, parts, static_cast<int>(count));
                SMX_LAUNCH_CHECK("k_norm_gradient_join");
            }
        });
    });
}

}  // extern "C"
