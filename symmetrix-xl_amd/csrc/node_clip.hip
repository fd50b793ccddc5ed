// The norm of many gradients together, and their clipping to a largest norm.
//
//   norm = scale * sqrt(sum of all squares)      out = g * scale * min(1, max_norm / norm)
//
// Bytes bound both: every gradient is read once for the norm and once more for the clipping.  Squares and sums are held in FP64, which
// the squares of no FP32 value leave and whose rate (one product-sum a value) stays below memory's; a square of FP32 would overflow
// from 2^64 on.  Tensors come in a table of kernel arguments, so nothing is copied to the card and a call may be captured;
// workgroups walk chunks of all of them, each keeps one sum, and every workgroup of the second kernel adds these up again in
// one order, so the second launch is the last.
#include <algorithm>
#include <cmath>
#include <vector>

#include "node_ops.hpp"

namespace smx {
namespace node {
namespace {

constexpr int kTensors = 96;      // of one launch: the table is of kernel arguments, of which there are 4 KB
constexpr int kChunk = 16384;     // values
constexpr int kTables = 1024;     // launches at most
constexpr int kParts = 2048;      // sums of the first kernel, of all launches (402 million bf16 values in 141 us, 149 with 1,024)
constexpr int kThreads = 256;

struct Tensors {
    const void* at[kTensors];
    void* out[kTensors];
    i64 count[kTensors];
    unsigned first[kTensors + 1];  // chunk of each
    std::uint8_t kind[kTensors], out_kind[kTensors];
    int tensors;
};
static_assert(sizeof(Tensors) <= 3584);

__device__ __forceinline__ int tensor_of(const Tensors& t, unsigned chunk) {
    int lo = 0, n = t.tensors;
    while (n > 1) {
        const int half = n / 2;
        if (t.first[lo + half] <= chunk) lo += half, n -= half;
        else n = half;
    }
    return lo;
}

// f(values, index, count) for packs of eight values of a chunk that are there whole, f with a count below eight at its end
template <class T, class F>
__device__ __forceinline__ void each_eight(const T* at, i64 n, F&& f) {
    constexpr int kAhead = 4;
    i64 c = 8 * threadIdx.x;
    for (; c + 8 * kThreads * (kAhead - 1) + 8 <= n; c += 8 * kThreads * kAhead) {
        Eight<T> e[kAhead];
#pragma unroll
        for (int q = 0; q < kAhead; ++q) e[q] = load_pack(at + c + 8 * kThreads * q, 0, 8);
#pragma unroll
        for (int q = 0; q < kAhead; ++q) f(e[q], c + 8 * kThreads * q, 8);
    }
    for (; c < n; c += 8 * kThreads) {
        const int left = n - c < 8 ? static_cast<int>(n - c) : 8;
        Eight<T> e = load_pack(at + c, 0, left);
        settle(e, 0, left);
        f(e, c, left);
    }
}

__device__ __forceinline__ double group_sum(double v, double (&room)[kThreads / 64]) {
    v = wave_sum<64>(v);
    if (threadIdx.x % 64 == 0) room[threadIdx.x / 64] = v;
    __syncthreads();
    v = room[0];
#pragma unroll
    for (int w = 1; w < kThreads / 64; ++w) v += room[w];
    return v;
}

// 402 million bf16 values in 120 tensors: 141 us, 5.7 TB/s, the rate of a read; 1.5 million FP32 ones in 14 tensors 4.5 us, of which the
// launch is most.
__global__ void __launch_bounds__(kThreads) k_norm_parts(Tensors t, double* __restrict__ parts) {
    __shared__ double room[kThreads / 64];
    double sum = 0.0;
    for (unsigned chunk = blockIdx.x; chunk < t.first[t.tensors]; chunk += gridDim.x) {
        const int i = tensor_of(t, chunk);
        const i64 from = static_cast<i64>(chunk - t.first[i]) * kChunk;
        const i64 n = t.count[i] - from < kChunk ? t.count[i] - from : kChunk;
        const auto go = [&](auto* at) {
            double s[8] = {};
            each_eight(at + from, n, [&](const auto& e, i64, int) {
#pragma unroll
                for (int q = 0; q < 8; ++q) s[q] = fma(static_cast<double>(e[q]), static_cast<double>(e[q]), s[q]);
            });
            sum += ((s[0] + s[1]) + (s[2] + s[3])) + ((s[4] + s[5]) + (s[6] + s[7]));
        };
        if (t.kind[i] == SMX_DTYPE_F32) go(static_cast<const float*>(t.at[i]));
        else if (t.kind[i] == SMX_DTYPE_BF16) go(static_cast<const bf16*>(t.at[i]));
        else go(static_cast<const f16*>(t.at[i]));
    }
    sum = group_sum(sum, room);
    if (threadIdx.x == 0) parts[blockIdx.x] = sum;
}

// The norm from the parts, the same in every workgroup.
__device__ __forceinline__ double norm_of(const double* parts, int count, float scale, double (&room)[kThreads / 64]) {
    double v = 0.0;
#pragma unroll
    for (int q = 0; q < kParts / kThreads; ++q) {
        const int p = q * kThreads + threadIdx.x;
        v += p < count ? parts[p] : 0.0;
    }
    return static_cast<double>(scale) * sqrt(group_sum(v, room));
}

__global__ void __launch_bounds__(kThreads) k_norm_join(const double* __restrict__ parts, int count, float scale,
                                                        float* __restrict__ norm) {
    __shared__ double room[kThreads / 64];
    const double v = norm_of(parts, count, scale, room);
    if (threadIdx.x == 0) *norm = static_cast<float>(v);
}

// out = at * by * 2^power: sixteen bytes of the outputs a lane, side by side for neighbouring lanes.
template <class T, class O>
__device__ __forceinline__ void scaled(const T* at, O* out, i64 n, float by, int power) {
    constexpr int N = 16 / sizeof(O), kAhead = 4;
    i64 c = N * static_cast<i64>(threadIdx.x);
    for (; c + N * kThreads * (kAhead - 1) + N <= n; c += N * kThreads * kAhead) {
        Pack<T, N> e[kAhead];
#pragma unroll
        for (int q = 0; q < kAhead; ++q) e[q] = *reinterpret_cast<const Pack<T, N>*>(at + c + N * kThreads * q);
#pragma unroll
        for (int q = 0; q < kAhead; ++q) {
            Pack<O, N> o;
#pragma unroll
            for (int i = 0; i < N; ++i) o.v[i] = static_cast<O>(__builtin_ldexpf(static_cast<float>(e[q].v[i]) * by, power));
            *reinterpret_cast<Pack<O, N>*>(out + c + N * kThreads * q) = o;
        }
    }
    for (; c < n; c += N * kThreads)
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (c + i < n) out[c + i] = static_cast<O>(__builtin_ldexpf(static_cast<float>(at[c + i]) * by, power));
}

// A chunk a workgroup, whose order the card's scheduler keeps even: 402 million values from bf16 to FP32 in 437 us, 5.5 TB/s (a
// copy 4.7; the cached end of the first kernel's reads helps).  The whole call 616 us, 684 in 2,048 workgroups of several chunks;
// stores that pass by the caches took 803.  1.5 million values 6.5 us.
__global__ void __launch_bounds__(kThreads) k_clip(Tensors t, const double* __restrict__ parts, int count, float scale,
                                                   float max_norm, float* __restrict__ norm) {
    __shared__ double room[kThreads / 64];
    const double total = norm_of(parts, count, scale, room);
    if (norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = static_cast<float>(total);
    // (a norm that is no number makes the factor none)
    const double factor = total <= max_norm ? scale : scale * (max_norm / total);
    // A factor that is a normal number of FP32 (no scale is more than one) is one product, rounded once.  A smaller one, of values
    // next to FP32's largest, is a significand in [0.5, 1) and a power of two, so that it keeps its bits: the products
    // may well be normal numbers.  A value that loses bits in the first of these two steps is 0 after the second.
    int power = 0;
    const float by = static_cast<float>(factor > 0.0 && factor < 0x1p-126 ? frexp(factor, &power) : factor);
    // The tensors come the last first, and a tensor's last chunk too: what was read last is still in the last cache (256 MB).
    const unsigned chunks = t.first[t.tensors];
    for (unsigned nth = blockIdx.x; nth < chunks; nth += gridDim.x) {
        const int i = tensor_of(t, nth);
        const unsigned chunk = t.first[i] + t.first[i + 1] - 1 - nth;
        const i64 from = static_cast<i64>(chunk - t.first[i]) * kChunk;
        const i64 n = t.count[i] - from < kChunk ? t.count[i] - from : kChunk;
        const bool whole = factor == 1.0;
        const auto go = [&](auto* at, auto* out) {
            if (whole && static_cast<const void*>(at) == out) return;  // values as they are, in place
            scaled(at + from, out + from, n, by, power);
        };
        const auto to = [&](auto* at) {
            if (t.out_kind[i] == SMX_DTYPE_F32) go(at, static_cast<float*>(t.out[i]));
            else if (t.out_kind[i] == SMX_DTYPE_BF16) go(at, static_cast<bf16*>(t.out[i]));
            else go(at, static_cast<f16*>(t.out[i]));
        };
        if (t.kind[i] == SMX_DTYPE_F32) to(static_cast<const float*>(t.at[i]));
        else if (t.kind[i] == SMX_DTYPE_BF16) to(static_cast<const bf16*>(t.at[i]));
        else to(static_cast<const f16*>(t.at[i]));
    }
}

struct List {
    const void* const* at;
    const i64* counts;
    const std::int32_t* dtypes;
    i64 tensors;
    void* const* out;
    const std::int32_t* out_dtypes;
};

i64 chunks_of(i64 values) { return (values + kChunk - 1) / kChunk; }

void check_list(const List& l, float scale) {
    require(l.tensors >= 0 && l.tensors <= (1 << 20), "the number of tensors must be in [0, 2^20]");
    require(l.tensors == 0 || (l.at && l.counts && l.dtypes), "the tensors' addresses, counts or types are NULL");
    require(scale > 0.0f && std::isfinite(scale), "scale must be positive and finite");
    for (i64 i = 0; i < l.tensors; ++i) {
        require(l.counts[i] >= 0 && l.counts[i] <= (1LL << 40), "a tensor's count must be in [0, 2^40]");
        require(l.dtypes[i] >= SMX_DTYPE_F32 && l.dtypes[i] <= SMX_DTYPE_F16, "unknown dtype code");
        require(l.counts[i] == 0 || l.at[i], "a tensor is NULL");
        require(aligned(l.at[i], static_cast<std::size_t>(size_of(l.dtypes[i]))), "a tensor is not aligned to its values");
    }
}

// Outputs do not overlap each other, nor a gradient that is not their own.
void check_outputs(const List& l) {
    struct Range {
        std::uintptr_t begin, end;
        i64 index;
    };
    std::vector<Range> ranges;
    ranges.reserve(static_cast<std::size_t>(l.tensors));
    for (i64 i = 0; i < l.tensors; ++i) {
        require(l.out_dtypes[i] >= SMX_DTYPE_F32 && l.out_dtypes[i] <= SMX_DTYPE_F16, "unknown dtype code");
        if (l.counts[i] == 0) continue;
        require(l.out[i], "an output is NULL");
        require(aligned(l.out[i], static_cast<std::size_t>(size_of(l.out_dtypes[i]))), "an output is not aligned to its values");
        const auto begin = reinterpret_cast<std::uintptr_t>(l.out[i]);
        ranges.push_back({begin, begin + static_cast<std::uintptr_t>(l.counts[i]) * static_cast<std::uintptr_t>(size_of(l.out_dtypes[i])), i});
    }
    std::sort(ranges.begin(), ranges.end(), [](const Range& a, const Range& b) { return a.begin < b.begin; });
    for (std::size_t i = 1; i < ranges.size(); ++i) require(ranges[i - 1].end <= ranges[i].begin, "two outputs overlap");
    for (i64 i = 0; i < l.tensors; ++i) {
        if (l.counts[i] == 0) continue;
        const auto begin = reinterpret_cast<std::uintptr_t>(l.at[i]);
        const auto end = begin + static_cast<std::uintptr_t>(l.counts[i]) * static_cast<std::uintptr_t>(size_of(l.dtypes[i]));
        auto r = std::upper_bound(ranges.begin(), ranges.end(), begin, [](std::uintptr_t v, const Range& q) { return v < q.end; });
        for (; r != ranges.end() && r->begin < end; ++r)
            require(r->index == i && r->begin == begin && l.dtypes[i] == l.out_dtypes[i],
                    "an output overlaps a gradient that is not its own in its own type");
    }
}

// f(table, chunks) for each launch's tensors, from the first tensor on or (`backwards`) from the last
template <class F>
void each_table(const List& l, F&& f, bool backwards = false) {
    Tensors t;
    i64 done = 0;
    while (done < l.tensors) {
        t.tensors = 0;
        i64 chunks = 0;
        for (; done < l.tensors && t.tensors < kTensors; ++done) {
            const i64 i = backwards ? l.tensors - 1 - done : done;
            if (l.counts[i] == 0) continue;
            const i64 more = chunks_of(l.counts[i]);
            if (chunks + more > (1LL << 31)) {
                require(t.tensors > 0, "a tensor is too large");
                break;
            }
            const int n = t.tensors++;
            t.at[n] = l.at[i], t.count[n] = l.counts[i], t.kind[n] = static_cast<std::uint8_t>(l.dtypes[i]);
            t.out[n] = l.out ? l.out[i] : nullptr;
            t.out_kind[n] = l.out ? static_cast<std::uint8_t>(l.out_dtypes[i]) : 0;
            t.first[n] = static_cast<unsigned>(chunks);
            chunks += more;
        }
        if (t.tensors == 0) return;
        t.first[t.tensors] = static_cast<unsigned>(chunks);
        f(t, chunks);
    }
}

// The first kernel over all tables; the number of its sums.
int launch_parts(const List& l, double* parts, hipStream_t stream) {
    i64 tables = 0;
    each_table(l, [&](const Tensors&, i64) { ++tables; });
    if (tables > kTables) throw std::domain_error("the gradients' norm takes up to 98304 tensors");
    const i64 most = tables > 0 ? kParts / tables : 0;
    int used = 0;
    each_table(l, [&](const Tensors& t, i64 chunks) {
        const int grid = static_cast<int>(chunks < most ? chunks : most);
        k_norm_parts<<<static_cast<unsigned>(grid), kThreads, 0, stream>>>(t, parts + used);
        SMX_LAUNCH_CHECK("k_norm_parts");
        used += grid;
    });
    return used;
}

}  // namespace
}  // namespace node
}  // namespace smx

using namespace smx;
using namespace smx::node;

extern "C" {

int64_t smx_gradient_norm_workspace(void) { return kParts * static_cast<i64>(sizeof(double)); }

int32_t smx_gradient_norm(const void* const* tensors, const int64_t* counts, const int32_t* dtypes, int64_t num_tensors, float scale,
                          float* norm, void* workspace, int64_t workspace_bytes, void* stream) {
    return guarded([&] {
        const List l{tensors, reinterpret_cast<const i64*>(counts), dtypes, num_tensors, nullptr, nullptr};
        check_list(l, scale);
        require(norm && aligned(norm, 4), "norm is NULL or not aligned");
        check_workspace(workspace, workspace_bytes, smx_gradient_norm_workspace());
        auto* const parts = static_cast<double*>(workspace);
        const int used = launch_parts(l, parts, static_cast<hipStream_t>(stream));
        k_norm_join<<<1, kThreads, 0, static_cast<hipStream_t>(stream)>>>(parts, used, scale, norm);
        SMX_LAUNCH_CHECK("k_norm_join");
    });
}

int32_t smx_clip_gradients(const void* const* tensors, const int64_t* counts, const int32_t* dtypes, int64_t num_tensors,
                           float max_norm, float scale, void* const* out, const int32_t* out_dtypes, float* norm, void* workspace,
                           int64_t workspace_bytes, void* stream) {
    return guarded([&] {
        const List l{tensors, reinterpret_cast<const i64*>(counts), dtypes, num_tensors, out, out_dtypes};
        check_list(l, scale);
        require(max_norm >= 0.0f, "max_norm must not be negative or NaN");
        require(num_tensors == 0 || (out && out_dtypes), "the outputs' addresses or types are NULL");
        check_outputs(l);
        require(norm && aligned(norm, 4), "norm is NULL or not aligned");
        check_workspace(workspace, workspace_bytes, smx_gradient_norm_workspace());
        auto* const parts = static_cast<double*>(workspace);
        const auto at = static_cast<hipStream_t>(stream);
        const int used = launch_parts(l, parts, at);
        if (used == 0) {
            k_norm_join<<<1, kThreads, 0, at>>>(parts, 0, scale, norm);
            SMX_LAUNCH_CHECK("k_norm_join");
            return;
        }
        float* first = norm;
        each_table(l, [&](const Tensors& t, i64 chunks) {
            const unsigned grid = static_cast<unsigned>(chunks < 16384 ? chunks : 16384);
            k_clip<<<grid, kThreads, 0, at>>>(t, parts, used, scale, max_norm, first);
            SMX_LAUNCH_CHECK("k_clip");
            first = nullptr;
        }, true);
    });
}

}  // extern "C"
