// Rows by kind: a stable order of the rows by their kind, and where each kind's rows begin in it.
//
// One counting pass, a kind a digit: tiles of rows are counted, and each tile places its rows by the counts of all tiles
// before it.  Waves rank 64 rows at a time with ballots, one for each bit of the kind, and keep counts of their own, so
// that they rank side by side and the order does not depend on which is first.  Up to kRows rows one workgroup does all.
#include "node_grouped.hpp"

namespace smx {
namespace node {
namespace {

constexpr int kWaves = 16, kThreads = 64 * kWaves;
constexpr int kPerLane = 2, kRows = kThreads * kPerLane;  // rows of a round

template <class I>
__device__ __forceinline__ int kind_of(const I* types, i64 t, int kinds) {
    const I z = types[t];
    return z >= 0 && static_cast<i64>(z) < kinds ? static_cast<int>(z) : kinds;
}

// A tile's counts of the kinds, by additions in LDS.  Waited for rather than bound by bytes: 131,072 rows in 2.7 us, of which
// the launch is most.
template <class I>
__global__ void __launch_bounds__(kThreads) k_group_count(const I* __restrict__ types, i64 rows, int kinds, i64 tile,
                                                          int* __restrict__ counts) {
    __shared__ int count[kMostKinds + 1];
    for (int d = threadIdx.x; d <= kinds; d += kThreads) count[d] = 0;
    __syncthreads();
    const i64 first = blockIdx.x * tile, last = first + tile < rows ? first + tile : rows;
    for (i64 t = first + threadIdx.x; t < last; t += kThreads) atomicAdd(&count[kind_of(types, t, kinds)], 1);
    __syncthreads();
    for (int d = threadIdx.x; d <= kinds; d += kThreads) counts[blockIdx.x * (kinds + 1LL) + d] = count[d];
}

// Sums of the threads before, of two numbers in one each: the workgroup's totals in `all`.
template <int N>
struct Sums {
    unsigned long long v[N];
};

template <int N>
__device__ __forceinline__ Sums<N> sum_before(const Sums<N>& of, unsigned long long (&room)[3][kWaves], Sums<N>& all) {
    const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
    Sums<N> sum = of;
#pragma unroll
    for (int o = 1; o < 64; o *= 2)
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const unsigned long long below = __shfl_up(sum.v[i], o);
            if (lane >= o) sum.v[i] += below;
        }
    __syncthreads();
    if (lane == 63)
#pragma unroll
        for (int i = 0; i < N; ++i) room[i][wave] = sum.v[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
        sum.v[i] -= of.v[i];
        all.v[i] = 0;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            if (w < wave) sum.v[i] += room[i][w];
            all.v[i] += room[i][w];
        }
    }
    return sum;
}

// BITS: of a kind; the waves' counts of all kinds are in LDS (147 KB of it at 13 bits, so kinds are 4,096 at most, and 8 and 10 bits
// leave room for more and shorter loops).  ONE: one workgroup, nothing was counted.
//
// Latency bounds it: reads of the counts, one scan over the kinds for offsets, present kinds and tiles of three sizes together, a round
// of ballots, and the stores.  135 rows of 89 kinds in 6.5 us, 131,071 of 1,009 in 13.9 us (1.5 MB of rows and order).
template <class I, int BITS, bool ONE>
__global__ void __launch_bounds__(kThreads) k_group_place(const I* __restrict__ types, i64 rows, int kinds, i64 tile,
                                                          const int* __restrict__ counts, int* __restrict__ plan) {
    constexpr int kDigits = BITS == 13 ? kMostKinds + 8 : 1 << BITS;
    // of a round: of each wave, then of the waves before; a kind's sixteen are 32 bytes
    __shared__ __attribute__((aligned(16))) std::uint16_t count[kDigits][kWaves];
    __shared__ int base[kDigits];
    __shared__ unsigned long long room[3][kWaves];
    __shared__ int most;  // rows of a kind
    if (threadIdx.x == 0) most = 0;
    const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
    int* const order = plan + plan_order(kinds);
    const i64 first = blockIdx.x * tile, last = first + tile < rows ? first + tile : rows;
    for (i64 at = first;; at += kRows) {
        // ranks
        for (int d = threadIdx.x; d < kWaves * kDigits / 8; d += kThreads) reinterpret_cast<uint4*>(count)[d] = uint4{0, 0, 0, 0};
        __syncthreads();
        int kind[kPerLane], rank[kPerLane];
        bool in[kPerLane];
#pragma unroll
        for (int k = 0; k < kPerLane; ++k) {
            const i64 t = at + wave * 64 * kPerLane + 64 * k + lane;
            in[k] = t < last;
            kind[k] = in[k] ? kind_of(types, t, kinds) : 0;
        }
#pragma unroll
        for (int k = 0; k < kPerLane; ++k) {
            unsigned long long same = __ballot(in[k]);
#pragma unroll
            for (int b = 0; b < BITS; ++b) {
                const unsigned long long w = __ballot(kind[k] >> b & 1);
                same &= kind[k] >> b & 1 ? w : ~w;
            }
            const int before = __popcll(same & ((1ull << lane) - 1));
            const int had = in[k] ? count[kind[k]][wave] : 0;
            rank[k] = had + before;
            __builtin_amdgcn_wave_barrier();
            if (in[k] && before == 0) count[kind[k]][wave] = static_cast<std::uint16_t>(had + __popcll(same));
            __builtin_amdgcn_wave_barrier();
        }
        __syncthreads();
        // the round's counts, and in the first round where each kind begins
        int total[(kDigits + kThreads - 1) / kThreads];
        Sums<3> carry{};
#pragma unroll
        for (int c = 0; c < (kDigits + kThreads - 1) / kThreads; ++c) {
            if (c * kThreads > kinds) break;
            const int d = c * kThreads + threadIdx.x;
            int sum = 0;
            if (d <= kinds) {
                uint4* const mine = reinterpret_cast<uint4*>(count[d]);
                uint4 w[2] = {mine[0], mine[1]};
                unsigned* const two = reinterpret_cast<unsigned*>(w);
#pragma unroll
                for (int i = 0; i < kWaves / 2; ++i) {
                    const unsigned lo = two[i] & 0xffffu, hi = two[i] >> 16;
                    two[i] = static_cast<unsigned>(sum) | (static_cast<unsigned>(sum) + lo) << 16;
                    sum += static_cast<int>(lo + hi);
                }
                mine[0] = w[0], mine[1] = w[1];
            }
            total[c] = sum;
            if (at > first) continue;
            int before = 0, all = 0;
            if constexpr (ONE) {
                all = sum;
            } else if (d <= kinds) {
#pragma unroll 32
                for (int b = 0; b < static_cast<int>(gridDim.x); ++b) {
                    const int n = counts[b * (kinds + 1LL) + d];
                    before += b < static_cast<int>(blockIdx.x) ? n : 0;
                    all += n;
                }
            }
            const unsigned long long seen = static_cast<unsigned long long>(all > 0) << 32 | static_cast<unsigned>(all);
            if (blockIdx.x > 0) {
                Sums<1> whole;
                const Sums<1> sums = sum_before(Sums<1>{seen}, room, whole);
                if (d <= kinds) base[d] = static_cast<int>((sums.v[0] + carry.v[0]) & 0xffffffffu) + before;
                carry.v[0] += whole.v[0];
                continue;
            }
            // tiles of 64 and 128 rows, and of 256
            const auto tiles = [&](int size) { return static_cast<unsigned>((all + size - 1) / size); };
            Sums<3> whole;
            Sums<3> sums = sum_before(Sums<3>{seen, static_cast<unsigned long long>(tiles(64)) << 32 | tiles(128), tiles(256)}, room, whole);
#pragma unroll
            for (int i = 0; i < 3; ++i) sums.v[i] += carry.v[i], carry.v[i] += whole.v[i];
            const int start = static_cast<int>(sums.v[0] & 0xffffffffu), index = static_cast<int>(sums.v[0] >> 32);
            int largest = d < kinds ? all : 0;
#pragma unroll
            for (int o = 1; o < 64; o *= 2) {
                const int other = __shfl_xor(largest, o);
                largest = other > largest ? other : largest;
            }
            if (lane == 0) atomicMax(&most, largest);
            if (d > kinds) continue;
            base[d] = start + before;
            plan[plan_offsets() + d] = start;
            if (all > 0) {
                plan[plan_present(kinds) + index] = d;
                plan[plan_start(kinds) + index] = start;
                plan[plan_tiles(kinds, 0) + index] = static_cast<int>(sums.v[1] >> 32);
                plan[plan_tiles(kinds, 1) + index] = static_cast<int>(sums.v[1] & 0xffffffffu);
                plan[plan_tiles(kinds, 2) + index] = static_cast<int>(sums.v[2]);
            }
        }
        __syncthreads();
        if (at == first && blockIdx.x == 0 && threadIdx.x == 0) {
            const int present = static_cast<int>(carry.v[0] >> 32);
            plan[0] = present;
            plan[1] = static_cast<int>(rows), plan[2] = kinds, plan[3] = most;
            plan[plan_start(kinds) + present] = static_cast<int>(rows);
            plan[plan_tiles(kinds, 0) + present] = static_cast<int>(carry.v[1] >> 32);
            plan[plan_tiles(kinds, 1) + present] = static_cast<int>(carry.v[1] & 0xffffffffu);
            plan[plan_tiles(kinds, 2) + present] = static_cast<int>(carry.v[2]);
            plan[plan_offsets() + kinds + 1] = static_cast<int>(rows);
        }
#pragma unroll
        for (int k = 0; k < kPerLane; ++k)
            if (in[k])
                order[base[kind[k]] + count[kind[k]][wave] + rank[k]] = static_cast<int>(at + wave * 64 * kPerLane + 64 * k + lane);
        if (at + kRows >= last) return;
        __syncthreads();
#pragma unroll
        for (int c = 0; c < (kDigits + kThreads - 1) / kThreads; ++c) {
            const int d = c * kThreads + threadIdx.x;
            if (d <= kinds) base[d] += total[c];
        }
    }
}

// Tiles of rows: each reads the counts of all, so no more than read 1 MB each, nor more than the card has units.
i64 tiles_of(i64 rows, i64 kinds) {
    i64 most = (1 << 18) / (kinds + 1);
    most = most < 16 ? 16 : most > kComputeUnits ? kComputeUnits : most;
    const i64 tiles = (rows + kRows - 1) / kRows;
    return tiles < most ? tiles : most;
}

template <class I>
void group(const I* types, i64 rows, int kinds, int* plan, int* counts, hipStream_t stream) {
    const i64 most = tiles_of(rows, kinds), tile = most > 1 ? ((rows + most - 1) / most + kRows - 1) / kRows * kRows : kRows;
    const unsigned tiles = rows > 0 ? static_cast<unsigned>((rows + tile - 1) / tile) : 1;
    const auto place = [&](auto bits) {
        constexpr int B = decltype(bits)::value;
        if (tiles == 1)
            k_group_place<I, B, true><<<1, kThreads, 0, stream>>>(types, rows, kinds, tile, counts, plan);
        else
            k_group_place<I, B, false><<<tiles, kThreads, 0, stream>>>(types, rows, kinds, tile, counts, plan);
        SMX_LAUNCH_CHECK("k_group_place");
    };
    if (tiles > 1) {
        k_group_count<I><<<tiles, kThreads, 0, stream>>>(types, rows, kinds, tile, counts);
        SMX_LAUNCH_CHECK("k_group_count");
    }
    using std::integral_constant;
    if (kinds < 1 << 8) place(integral_constant<int, 8>{});
    else if (kinds < 1 << 10) place(integral_constant<int, 10>{});
    else place(integral_constant<int, 13>{});
}

bool sizes_ok(i64 rows, i64 kinds) { return rows >= 0 && rows <= (1LL << 30) && kinds >= 1 && kinds <= kMostKinds; }

}  // namespace
}  // namespace node
}  // namespace smx

using namespace smx;
using namespace smx::node;

extern "C" {

int64_t smx_group_plan_order(int64_t num_types) { return num_types >= 1 ? 4 * plan_order(num_types) : 0; }

int64_t smx_group_plan_bytes(int64_t rows, int64_t num_types) {
    return sizes_ok(rows, num_types) ? 4 * (plan_order(num_types) + rows) : 0;
}

int64_t smx_group_rows_workspace(int64_t rows, int64_t num_types) {
    if (!sizes_ok(rows, num_types) || rows <= kRows) return 0;
    return 4 * tiles_of(rows, num_types) * (num_types + 1);
}

int32_t smx_group_rows(const void* types, int32_t types_are_64bit, int64_t rows, int64_t num_types, void* plan,
                       int64_t plan_bytes, void* workspace, int64_t workspace_bytes, void* stream) {
    return guarded([&] {
        require(rows >= 0 && rows <= (1LL << 30), "rows must be in [0, 2^30]");
        require(num_types >= 1, "there must be a kind at least");
        if (num_types > kMostKinds) throw std::domain_error("rows are grouped by up to 4096 kinds");
        require(rows == 0 || types, "types is NULL");
        require(aligned(types, types_are_64bit ? 8 : 4), "types is not aligned to its values");
        require(plan && aligned(plan, 16), "the plan is NULL or not 16-byte aligned");
        require(plan_bytes >= smx_group_plan_bytes(rows, num_types), "the plan is too small");
        check_workspace(workspace, workspace_bytes, smx_group_rows_workspace(rows, num_types));
        const int kinds = static_cast<int>(num_types);
        if (types_are_64bit)
            group(static_cast<const long long*>(types), rows, kinds, static_cast<int*>(plan), static_cast<int*>(workspace),
                  static_cast<hipStream_t>(stream));
        else
            group(static_cast<const int*>(types), rows, kinds, static_cast<int*>(plan), static_cast<int*>(workspace),
                  static_cast<hipStream_t>(stream));
    });
}

}  // extern "C"
