// Products of rows with the weights of their kind, and their gradients: kernels by value type, instantiated by
// node_grouped_*.hip, launched by node_grouped.hip.
//
//   forward   y_t  = W_z(t) x_t            a tile: up to BM rows of one kind, gathered by the plan, times BN outputs
//   by x      dx_t = W_z(t)^T g_t          the same with the weights read across their rows
//   by W      dW_z = sum over t of g_t x_t^T    a tile: BM x BN of one kind's weights, a run of its rows summed
//
// Sizes of the kinds are known to the device alone, so a launch has as many workgroups as the card holds, which walk the
// tiles that the plan gives.  Tile u of the rows: with the kinds that have rows in order, p the p-th and s(p) its first sorted row, kind
// p's tiles are numbered from p + s(p) / BM on.  It has at most 1 + s(p + 1) / BM - s(p) / BM of them, so numbers do not
// meet, and at most one a kind is not used.  Likewise the runs of a kind's rows in the weights' gradient, cut at multiples of
// `run` sorted rows: kind z's are numbered from z + offset(z) / run on.
#pragma once

#include "node_tiles.hpp"

namespace smx {
namespace node {

// ---- the plan (node_group.hip), in ints: the number of kinds that have rows; offsets; these kinds and their first
// sorted rows; the order.  Rows of no kind are kind `kinds`. ----

constexpr i64 kMostKinds = 4096;
constexpr i64 kMostRows = (1LL << 31) - 65536;

inline __host__ __device__ i64 plan_room(i64 kinds) { return (kinds + 5) / 4 * 4; }
inline __host__ __device__ i64 plan_offsets() { return 4; }
inline __host__ __device__ i64 plan_present(i64 kinds) { return 4 + plan_room(kinds); }
inline __host__ __device__ i64 plan_start(i64 kinds) { return 4 + 2 * plan_room(kinds); }
inline __host__ __device__ i64 plan_order(i64 kinds) { return 4 + 3 * plan_room(kinds); }

enum class Way { Forward, ByRows, ByWeights };

template <class T, class O>
struct Grouped {
    const T* a;  // x; the gradient of y in both gradients
    i64 a_stride;
    const T* b;  // the weights; x in the gradient by them
    i64 b_stride, b_kind;
    O* out;
    i64 out_stride, out_kind;
    const int* plan;
    int tokens, kinds;
    int m;  // by W: rows of a kind's weights
    int n;  // columns of out
    int k;  // summed (by W: the rows are)
    int tiles_m, tiles_n;
    int run, units;   // by W
    float* partial;  // by W, [2 per run][m][n], where kinds may be cut
};

// the last of the `count` ascending keys (key(0) <= u) that is <= u; by a whole wave
template <class F>
__device__ __forceinline__ int last_up_to(int u, int count, F&& key) {
    const int lane = threadIdx.x % 64;
    int first = 0;
    while (count > 1) {
        const int hop = (count + 63) / 64, at = lane * hop;
        const bool in = at < count && key(first + (at < count ? at : 0)) <= u;
        const int far = (__popcll(__ballot(in)) - 1) * hop;
        first += far;
        count = hop < count - far ? hop : count - far;
    }
    return __builtin_amdgcn_readfirstlane(first);
}

// Four neighbouring outputs from column j on.
template <class O>
__device__ __forceinline__ void store_outputs(O* row, int j, int n, acc4 v) {
    if (j + 4 <= n) {
        Pack<O, 4> o;
#pragma unroll
        for (int q = 0; q < 4; ++q) o.v[q] = static_cast<O>(v[q]);
        *reinterpret_cast<Pack<O, 4>*>(row + j) = o;
    } else {
#pragma unroll
        for (int q = 0; q < 4; ++q)
            if (j + q < n) row[j + q] = static_cast<O>(apart(v[q]));
    }
}

template <class T, class O, Way WAY, bool DIRECT, int BM, int BN, int WM, int WN>
__global__ void __launch_bounds__(64 * WM * WN, BM + BN > 256 ? 1 : 2) k_grouped_tiles(Grouped<T, O> p) {
    constexpr Lie LA = WAY == Way::ByWeights ? Lie::Columns : Lie::Rows, LB = WAY == Way::Forward ? Lie::Rows : Lie::Columns;
    using A = Step<T, LA, BM>;
    using B = Step<T, LB, BN>;
    constexpr int WAVES = WM * WN, NA = A::kPieces / 64 / WAVES, NB = B::kPieces / 64 / WAVES, MF = BM / WM / 16,
                  NF = BN / WN / 16, kPer = 16 / static_cast<int>(sizeof(T));
    constexpr unsigned kStage = (BM + BN) * kStepBytes;
    static_assert(A::kPieces % (64 * WAVES) == 0 && B::kPieces % (64 * WAVES) == 0);
    static_assert(WAY != Way::ByWeights || BM == BN);
    __shared__ __attribute__((aligned(1024))) std::uint8_t lds[2 * kStage];
    const unsigned lds0 = static_cast<unsigned>(reinterpret_cast<std::uintptr_t>((__attribute__((address_space(3))) std::uint8_t*)lds));
    const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const int wm = wave / WN * (BM / WM), wn = wave % WN * (BN / WN);
    const int* const order = p.plan + plan_order(p.kinds);
    const int present = WAY == Way::ByWeights ? 0 : p.plan[0];
    const int units = WAY == Way::ByWeights ? p.units : present + p.tokens / BM;
    const int tiles = units * p.tiles_m * p.tiles_n;

    // the tile whose steps are being read
    struct Tile {
        int row0, rows;  // sorted rows: of the tile, or of the run
        int i0, j0;
        int kind, steps, slot;  // slot: of the partial sums, or -1
    } next;
    const T* at_a[NA];  // Rows: where the lane's pieces of the first step are
    const T* at_b[NB];
    int id_a[NA];  // Columns of gathered rows: the rows of the step to come (a's and b's are the same)
    const auto steps_of = [](int k) { return (k + A::kValues - 1) / A::kValues; };
    const auto rows_of_step = [&](int s) {  // by W: asks for the ids of a step's rows, -1 past the end
#pragma unroll
        for (int q = 0; q < NA; ++q) {
            const int r = s * A::kValues + A::row_at((wave + WAVES * q) * 64 + lane);
            id_a[q] = r < next.rows ? order[next.row0 + r] : -1;
        }
    };
    const auto turn_to = [&](int turn) {
        const int id = xcd_remap(turn, tiles);
        if constexpr (WAY == Way::ByWeights) {
            const int per = p.tiles_m * p.tiles_n, u = id / per, in = id % per;
            const int* const offsets = p.plan + plan_offsets();
            next.kind = last_up_to(u, p.kinds, [&](int z) { return z + offsets[z] / p.run; });
            next.i0 = in % p.tiles_m * BM, next.j0 = in / p.tiles_m * BN;
            const int begin = offsets[next.kind], end = offsets[next.kind + 1], run = u - next.kind;
            next.slot = -1, next.rows = 0, next.steps = 0, next.row0 = begin;
            if (begin == end) return run == begin / p.run;
            if (run > (end - 1) / p.run) return false;
            const int first = run * p.run, last = first + p.run;
            if (begin < first) next.slot = 2 * run;
            else if (end > last) next.slot = 2 * run + 1;
            next.row0 = begin > first ? begin : first;
            next.rows = (end < last ? end : last) - next.row0;
            next.steps = steps_of(next.rows);
            rows_of_step(0);
        } else {
            // bands of four units, each column by column: neighbours share rows and weights in an XCD's L2
            const int band = id / (4 * p.tiles_n), in = id % (4 * p.tiles_n);
            const int high = units - 4 * band < 4 ? units - 4 * band : 4, u = 4 * band + in % high;
            const int* const start = p.plan + plan_start(p.kinds);
            const int at = last_up_to(u, present, [&](int q) { return q + start[q] / BM; });
            next.row0 = start[at] + (u - at - start[at] / BM) * BM;
            next.rows = start[at + 1] - next.row0 < BM ? start[at + 1] - next.row0 : BM;
            next.kind = p.plan[plan_present(p.kinds) + at];
            next.j0 = in / high * BN, next.i0 = 0;
            next.steps = next.kind == p.kinds ? 0 : steps_of(p.k);
            if (next.rows <= 0) return false;
            if (next.steps == 0) return true;
#pragma unroll
            for (int q = 0; q < NA; ++q) {
                const int e = (wave + WAVES * q) * 64 + lane, r = A::row_at(e);
                at_a[q] = p.a + order[next.row0 + (r < next.rows ? r : next.rows - 1)] * p.a_stride;
            }
            const T* const w = p.b + next.kind * p.b_kind;
#pragma unroll
            for (int q = 0; q < NB; ++q) {
                const int r = B::row_at((wave + WAVES * q) * 64 + lane);
                if constexpr (LB == Lie::Rows)
                    at_b[q] = w + (next.j0 + r < p.n ? next.j0 + r : p.n - 1) * p.b_stride;
                else
                    at_b[q] = w + r * p.b_stride;
            }
        }
        return true;
    };
    // (row and column of a's and b's pieces in memory; rows of no one are NULL)
    const auto piece_a = [&](int q, int s, const T*& row, i64& c, i64& cols) {
        const int piece = A::piece_at((wave + WAVES * q) * 64 + lane);
        if constexpr (LA == Lie::Rows) {
            row = at_a[q], c = static_cast<i64>(s) * A::kValues + piece * kPer, cols = p.k;
        } else {
            row = id_a[q] < 0 ? nullptr : p.a + id_a[q] * p.a_stride;
            c = next.i0 + piece * kPer, cols = p.m;
        }
    };
    const auto piece_b = [&](int q, int s, const T*& row, i64& c, i64& cols) {
        const int e = (wave + WAVES * q) * 64 + lane, piece = B::piece_at(e);
        if constexpr (LB == Lie::Rows) {
            row = at_b[q], c = static_cast<i64>(s) * B::kValues + piece * kPer, cols = p.k;
        } else if constexpr (WAY == Way::ByRows) {
            const int r = s * B::kValues + B::row_at(e);
            row = r < p.k ? at_b[q] + static_cast<i64>(s) * B::kValues * p.b_stride : nullptr;
            c = next.j0 + piece * kPer, cols = p.n;
        } else {
            row = id_a[q] < 0 ? nullptr : p.b + id_a[q] * p.b_stride;
            c = next.j0 + piece * kPer, cols = p.n;
        }
    };
    i32x4 held_a[DIRECT ? 1 : NA], held_b[DIRECT ? 1 : NB];
    // asks for step s of the tile `next`; DIRECT: into the slot, else into registers, which keep() brings there
    const auto stage = [&](int s, int slot) {
        const unsigned to = __builtin_amdgcn_readfirstlane(lds0 + slot * kStage);
        const T* row;
        i64 c, cols;
#pragma unroll
        for (int q = 0; q < NA; ++q) {
            piece_a(q, s, row, c, cols);
            if constexpr (DIRECT)
                fetch(row && c < cols ? static_cast<const void*>(row + c) : kNothing, to + (wave + WAVES * q) * 1024);
            else
                held_a[q] = row ? settle_piece<T>(load_piece(row, c, cols), c, cols) : i32x4{0, 0, 0, 0};
        }
#pragma unroll
        for (int q = 0; q < NB; ++q) {
            piece_b(q, s, row, c, cols);
            if constexpr (DIRECT)
                fetch(row && c < cols ? static_cast<const void*>(row + c) : kNothing,
                      to + BM * kStepBytes + (wave + WAVES * q) * 1024);
            else
                held_b[q] = row ? settle_piece<T>(load_piece(row, c, cols), c, cols) : i32x4{0, 0, 0, 0};
        }
        if constexpr (WAY == Way::ByWeights)
            if (s + 1 < next.steps) rows_of_step(s + 1);
    };
    const auto keep = [&](int slot) {
        if constexpr (!DIRECT) {
            std::uint8_t* const to = lds + slot * kStage + lane * 16;
#pragma unroll
            for (int q = 0; q < NA; ++q) *reinterpret_cast<i32x4*>(to + (wave + WAVES * q) * 1024) = held_a[q];
#pragma unroll
            for (int q = 0; q < NB; ++q)
                *reinterpret_cast<i32x4*>(to + BM * kStepBytes + (wave + WAVES * q) * 1024) = held_b[q];
        }
    };

    int slot = 0, turn = blockIdx.x;
    const auto advance = [&](int to) {  // to the next tile that is one, its first step into slot `to`
        while (turn < tiles && !turn_to(turn)) turn += gridDim.x;
        if (turn < tiles && next.steps > 0) stage(0, to);
    };
    advance(0);
    if (turn < tiles && next.steps > 0) keep(0);
    while (turn < tiles) {
        const Tile now = next;
        acc4 acc[MF][NF];
#pragma unroll
        for (int f = 0; f < MF; ++f)
#pragma unroll
            for (int g = 0; g < NF; ++g) acc[f][g] = acc4{0.0f, 0.0f, 0.0f, 0.0f};
        for (int s = 0; s < now.steps; ++s) {
            if constexpr (DIRECT) arrived();
            __syncthreads();  // the step is there, and all have read the one before
            const std::uint8_t* const tile = lds + slot * kStage;
            slot ^= 1;
            Fragment<T> vb[NF];
#pragma unroll
            for (int g = 0; g < NF; ++g) vb[g] = B::read(tile + BM * kStepBytes, wn + 16 * g, lane);
            if (s + 1 < now.steps) {
                stage(s + 1, slot);
            } else {
                turn += gridDim.x;
                advance(slot);
            }
#pragma unroll
            for (int f = 0; f < MF; ++f) {
                const Fragment<T> va = A::read(tile, wm + 16 * f, lane);
#pragma unroll
                for (int g = 0; g < NF; ++g) acc[f][g] = Fragment<T>::multiply(vb[g], va, acc[f][g]);
            }
            if (s + 1 < now.steps || (turn < tiles && next.steps > 0)) keep(slot);
        }
        if (now.steps == 0) {  // zeros: nothing was read
            turn += gridDim.x;
            advance(slot);
            if (turn < tiles && next.steps > 0) keep(slot);
        }
        settle_products();
        const int j0 = now.j0 + wn;
#pragma unroll
        for (int f = 0; f < MF; ++f) {
            const int i = wm + 16 * f + lane % 16;
            if constexpr (WAY == Way::ByWeights) {
                if (now.i0 + i >= p.m) continue;
                if (now.slot >= 0) {
                    float* const row = p.partial + (static_cast<i64>(now.slot) * p.m + now.i0 + i) * p.n;
#pragma unroll
                    for (int g = 0; g < NF; ++g) store_outputs(row, j0 + 16 * g + 4 * (lane / 16), p.n, acc[f][g]);
                } else {
                    O* const row = p.out + now.kind * p.out_kind + (now.i0 + i) * p.out_stride;
#pragma unroll
                    for (int g = 0; g < NF; ++g) store_outputs(row, j0 + 16 * g + 4 * (lane / 16), p.n, acc[f][g]);
                }
            } else {
                if (i >= now.rows) continue;
                O* const row = p.out + order[now.row0 + i] * p.out_stride;
#pragma unroll
                for (int g = 0; g < NF; ++g) store_outputs(row, j0 + 16 * g + 4 * (lane / 16), p.n, acc[f][g]);
            }
        }
    }
}

// The sums of kinds whose rows are cut: a workgroup row for each cut, which joins, in order, the runs of the kind that it
// is the first cut of.
template <class O>
__global__ void __launch_bounds__(256) k_grouped_join(const float* __restrict__ partial, const int* __restrict__ plan, int kinds,
                                                      int run, int m, int n, O* __restrict__ out, i64 out_stride, i64 out_kind) {
    const int cut = blockIdx.y + 1;
    const int* const offsets = plan + plan_offsets();
    if (cut * run >= offsets[kinds]) return;
    // (of kinds without rows at the cut itself, the last: it is the one whose rows follow)
    const int kind = last_up_to(cut * run, kinds, [&](int z) { return offsets[z]; });
    const int begin = offsets[kind], end = offsets[kind + 1], first = begin / run, last = (end - 1) / run;
    if (begin >= cut * run || first + 1 != cut) return;
    const i64 size = static_cast<i64>(m) * n;
    for (i64 e = static_cast<i64>(blockIdx.x) * 256 + threadIdx.x; e < size; e += static_cast<i64>(gridDim.x) * 256) {
        float sum = partial[(2 * first + 1) * size + e];
        for (int r = cut; r <= last; ++r) sum += partial[2 * r * size + e];
        out[kind * out_kind + e / n * out_stride + e % n] = static_cast<O>(sum);
    }
}

// Up to 16 rows of a kind: 16 NF outputs a workgroup, for kinds of few rows, whose weights are read once for all of them.
template <class T, class O, bool DIRECT, int NF, int KS>
__global__ void __launch_bounds__(64 * KS) k_grouped_rows(Grouped<T, O> p) {
    __shared__ FewRoom<T, NF, KS> room;
    const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const int present = p.plan[0], u = blockIdx.x / p.tiles_n, j0 = blockIdx.x % p.tiles_n * 16 * NF;
    if (u >= present + p.tokens / 16) return;
    const int* const start = p.plan + plan_start(p.kinds);
    const int* const order = p.plan + plan_order(p.kinds);
    const int at = last_up_to(u, present, [&](int q) { return q + start[q] / 16; });
    const int row0 = start[at] + (u - at - start[at] / 16) * 16, kind = p.plan[plan_present(p.kinds) + at];
    const int rows = start[at + 1] - row0 < 16 ? start[at + 1] - row0 : 16, row = lane % 16;
    if (rows <= 0) return;
    const int id = order[row0 + (row < rows ? row : rows - 1)];
    acc4 sum{0.0f, 0.0f, 0.0f, 0.0f};
    if (kind < p.kinds) {
        const T* b[NF];
#pragma unroll
        for (int g = 0; g < NF; ++g) {
            const int j = j0 + 16 * g + row;
            b[g] = p.b + kind * p.b_kind + (j < p.n ? j : p.n - 1) * p.b_stride;
        }
        sum = few_rows<T, DIRECT, NF, KS>(p.a + id * p.a_stride, b, p.k, room);
    }
    if (wave >= NF || row >= rows) return;
    store_outputs(p.out + id * p.out_stride, j0 + 16 * wave + 4 * (lane / 16), p.n, sum);
}

// How a call is cut (node_grouped.hip).
struct Cut {
    int tile;  // 256, 128, 64, or 16: k_grouped_rows
    bool direct;
    int units;  // of 16 rows, at most
};

template <class T, class O>
void launch_grouped(const Grouped<T, O>& p, Way way, const Cut& cut, hipStream_t stream) {
    const auto tiles = [&](auto w) {
        constexpr Way W = decltype(w)::value;
        if (!cut.direct) {
            k_grouped_tiles<T, O, W, false, 128, 128, 2, 2><<<2 * kComputeUnits, 256, 0, stream>>>(p);
        } else if (cut.tile == 256) {
            k_grouped_tiles<T, O, W, true, 256, 256, 2, 4><<<kComputeUnits, 512, 0, stream>>>(p);
        } else if (cut.tile == 128) {
            k_grouped_tiles<T, O, W, true, 128, 128, 2, 2><<<2 * kComputeUnits, 256, 0, stream>>>(p);
        } else {
            k_grouped_tiles<T, O, W, true, 64, 64, 2, 2><<<4 * kComputeUnits, 256, 0, stream>>>(p);
        }
        SMX_LAUNCH_CHECK("k_grouped_tiles");
    };
    using std::integral_constant;
    if (way == Way::ByRows) return tiles(integral_constant<Way, Way::ByRows>{});
    if (way == Way::ByWeights) return tiles(integral_constant<Way, Way::ByWeights>{});
    if (cut.tile != 16) return tiles(integral_constant<Way, Way::Forward>{});
    const unsigned grid = static_cast<unsigned>(cut.units) * static_cast<unsigned>(p.tiles_n);
    if (cut.direct)
        k_grouped_rows<T, O, true, 1, 8><<<grid, 512, 0, stream>>>(p);
    else
        k_grouped_rows<T, O, false, 1, 8><<<grid, 512, 0, stream>>>(p);
    SMX_LAUNCH_CHECK("k_grouped_rows");
}

}  // namespace node
}  // namespace smx
