// Products of rows with the weights of their kind, and their gradients: kernels by value type, instantiated by
// node_grouped_*.hip, launched by node_grouped.hip.
//
//   forward   y_t  = W_z(t) x_t            a tile: up to BM rows of one kind, gathered by the plan, times BN outputs
//   by x      dx_t = W_z(t)^T g_t          the same with the weights read across their rows
//   by W      dW_z = sum over t of g_t x_t^T    a tile: BM x BN of one kind's weights, a run of its rows summed
//
// Sizes of the kinds are known to the device alone, so a launch has as many workgroups as the card holds, which walk the tiles that
// the plan gives.  The runs of a kind's rows in the weights' gradient are cut at multiples of `run` sorted rows: kind z's are
// numbered from z + offset(z) / run on, of which it has at most 1 + offset(z + 1) / run - offset(z) / run.
#pragma once

#include <type_traits>

#include "node_tiles.hpp"

namespace smx {
namespace node {

// ---- the plan (node_group.hip), in ints: the number of kinds that have rows, that of all rows, of
// kinds and of the rows of the largest; offsets; these kinds, their first sorted rows
// and first tiles of 64, 128 and 256 rows; the order.  Rows of no kind are kind `kinds`. ----

constexpr i64 kMostKinds = 4096;

inline __host__ __device__ i64 plan_room(i64 kinds) { return (kinds + 5) / 4 * 4; }
inline __host__ __device__ i64 plan_offsets() { return 4; }
inline __host__ __device__ i64 plan_present(i64 kinds) { return 4 + plan_room(kinds); }
inline __host__ __device__ i64 plan_start(i64 kinds) { return 4 + 2 * plan_room(kinds); }
// the first tile of each of these kinds, and the number of tiles, where tiles have 64 << size rows
inline __host__ __device__ i64 plan_tiles(i64 kinds, int size) { return 4 + (3 + size) * plan_room(kinds); }
inline __host__ __device__ i64 plan_order(i64 kinds) { return 4 + 6 * plan_room(kinds); }

// whether a plan is of so many rows and kinds: nothing is read or written by another
__device__ __forceinline__ bool plan_fits(const int* plan, int rows, int kinds) { return plan[1] == rows && plan[2] == kinds; }

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
    int round, least;  // by W: units that the card holds at once, and the least run (0: kinds are not cut)
    float* partial;  // by W, [2 per run][m][n], where kinds may be cut
};

// Rows summed together in the weights' gradient, from the kinds' sizes, which the device has: a kind in one run where that takes no
// longer than a round or two of runs that fill the card, whose parts have to be joined (about 500 rows' time).  20,000 rows of 10 kinds
// are not cut, 30,000 of 2 in 59 runs.
__device__ __forceinline__ int run_of(const int* plan, int tokens, int round, int least) {
    const int count = plan[0], most = plan[3], whole = tokens + 1;
    if (least == 0) return whole;
    int run = whole;
    i64 best = static_cast<i64>((count + round - 1) / round) * most;
    for (int r = 1; r <= 2; ++r) {
        const int units = r * round - count;
        if (units <= 0) continue;
        int each = ((tokens + units - 1) / units + 63) / 64 * 64;
        each = each < least ? least : each;
        const i64 cost = static_cast<i64>(r) * each + 512;
        if (each < most && cost < best) best = cost, run = each;
    }
    return run;
}

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

// Eight neighbouring outputs of two bytes from column j on.
template <class O>
__device__ __forceinline__ void store_piece(O* row, int j, int n, i32x4 v) {
    struct __attribute__((packed, aligned(2))) Words {
        i32x4 w;
    };
    if (j + 8 <= n) {
        reinterpret_cast<Words*>(row + j)->w = v;
        return;
    }
    asm volatile("" : "+v"(v));  // (apart from the whole store)
#pragma unroll
    for (int q = 0; q < 8; ++q)
        if (j + q < n) row[j + q] = __builtin_bit_cast(O, static_cast<std::uint16_t>(static_cast<unsigned>(v[q / 2]) >> (16 * (q % 2))));
}

// Where a workgroup is: the tile that comes next, found while the one before is multiplied.  Up to 64 kinds are kept in
// the lanes of each wave, so that a tile is found without a read; more are looked up.
template <class T, class O, Way WAY, int BM, int BN>
struct Walk {
    const Grouped<T, O>* of;
    const int* order;
    int count, units, tiles, turn, run;
    bool even;  // by W: runs are of about one length
    int base_of, first_of, end_of, kind_of;  // of the lane's kind
    int row0, rows, i0, j0, kind, slot;  // of the tile: sorted rows; columns of out (by W: rows too); the partial sums' place, or -1

    __device__ __forceinline__ explicit Walk(const Grouped<T, O>& p) : of(&p), order(p.plan + plan_order(p.kinds)), turn(blockIdx.x) {
        const int lane = threadIdx.x % 64;
        count = run = units = tiles = 0, even = false;
        base_of = first_of = end_of = kind_of = 0;
        if (!__builtin_amdgcn_readfirstlane(plan_fits(p.plan, p.tokens, p.kinds))) return;
        count = __builtin_amdgcn_readfirstlane(WAY == Way::ByWeights ? p.kinds : p.plan[0]);
        if constexpr (WAY == Way::ByWeights) {
            run = __builtin_amdgcn_readfirstlane(run_of(p.plan, p.tokens, p.round, p.least));
            even = p.tiles_m * p.tiles_n <= 64 &&
                   __builtin_amdgcn_readfirstlane(run <= p.tokens ||
                                                  static_cast<i64>(p.plan[3]) * p.plan[0] <= 3 * (static_cast<i64>(p.tokens) / 2));
        }
        const int at = lane < count ? lane : count - 1;
        base_of = base(at), first_of = starts()[at], end_of = starts()[at + 1];
        kind_of = WAY == Way::ByWeights ? at : p.plan[plan_present(p.kinds) + at];
        units = __builtin_amdgcn_readfirstlane(WAY == Way::ByWeights ? p.kinds + p.tokens / run : base(count));
        tiles = units * p.tiles_m * p.tiles_n;
    }
    __device__ __forceinline__ const int* starts() const {
        const Grouped<T, O>& p = *of;
        return p.plan + (WAY == Way::ByWeights ? plan_offsets() : plan_start(p.kinds));
    }
    // the first unit of the q-th kind
    __device__ __forceinline__ int base(int q) const {
        const Grouped<T, O>& p = *of;
        if constexpr (WAY == Way::ByWeights) return q + starts()[q] / run;
        return p.plan[plan_tiles(p.kinds, BM == 64 ? 0 : BM == 128 ? 1 : 2) + q];
    }
    // the kind of unit u: its index, first unit, first and last sorted row and number
    __device__ __forceinline__ void find(int u, int& at, int& first, int& begin, int& end) {
        const Grouped<T, O>& p = *of;
        if (count <= 64) {
            const int lane = threadIdx.x % 64;
            at = __popcll(__ballot(lane < count && base_of <= u)) - 1;
            first = __builtin_amdgcn_readlane(base_of, at), kind = __builtin_amdgcn_readlane(kind_of, at);
            begin = __builtin_amdgcn_readlane(first_of, at), end = __builtin_amdgcn_readlane(end_of, at);
        } else {
            at = last_up_to(u, count, [&](int q) { return base(q); });
            first = base(at), begin = starts()[at], end = starts()[at + 1];
            kind = WAY == Way::ByWeights ? at : p.plan[plan_present(p.kinds) + at];
        }
    }
    // 0: no tile; 1: one to be summed; 2: one of zeros
    __device__ __forceinline__ int look() {
        const Grouped<T, O>& p = *of;
        int at, first, begin, end;
        if constexpr (WAY == Way::ByWeights) {
            // Tiles in bands of four.  Runs of about one length and few tiles go to an XCD each, which then reads their rows once (20,000 x 512
            // x 1,024 of ten types 68 us, 72 else; of 64 types with 128 tiles each 964 and 897); otherwise all XCDs are on one run at a time.
            const int per = p.tiles_m * p.tiles_n, all = xcd_remap(turn, tiles);
            const int u = even ? all / per : turn / per, id = even ? all % per : xcd_remap(turn % per, per);
            find(u, at, first, begin, end);
            const int band = id / (4 * p.tiles_n), in = id % (4 * p.tiles_n);
            const int high = p.tiles_m - 4 * band < 4 ? p.tiles_m - 4 * band : 4;
            i0 = (4 * band + in % high) * BM, j0 = in / high * BN;
            const int nth = u - at;
            slot = -1, rows = 0, row0 = begin;
            if (begin == end) return nth == begin / run ? 2 : 0;
            if (nth > (end - 1) / run) return 0;
            const int from = nth * run, to = from + run;
            if (begin < from) slot = 2 * nth;
            else if (end > to) slot = 2 * nth + 1;
            row0 = begin > from ? begin : from;
            rows = (end < to ? end : to) - row0;
            return 1;
        } else {
            // bands of four units, each column by column: neighbours share rows and weights in an XCD's L2
            const int id = xcd_remap(turn, tiles);
            const int band = id / (4 * p.tiles_n), in = id % (4 * p.tiles_n);
            const int high = units - 4 * band < 4 ? units - 4 * band : 4, u = 4 * band + in % high;
            find(u, at, first, begin, end);
            // the kind's rows in as many tiles as it takes, of one height: a tile costs what its rows' products do, and reading the
            // weights again for a few rows would cost nearly as much as for all (64 kinds of about 512 rows, 2,048 x
            // 4,096: 720 us, 754 in tiles of 256 and what is left)
            const int tiles_of = (end - begin + BM - 1) / BM, each = ((end - begin + tiles_of - 1) / tiles_of + 15) / 16 * 16;
            row0 = begin + (u - first) * each;
            rows = end - row0 < each ? end - row0 : each;
            j0 = in / high * BN, i0 = 0, slot = -1;
            return kind == p.kinds || p.k == 0 ? 2 : 1;
        }
    }
    // the outputs' row i of the tile
    __device__ __forceinline__ O* out_row(int i) const {
        const Grouped<T, O>& p = *of;
        if constexpr (WAY == Way::ByWeights)
            return p.out + kind * p.out_kind + (i0 + i) * p.out_stride;
        else
            return p.out + order[row0 + i] * p.out_stride;
    }
    __device__ __forceinline__ int out_rows() const {
        const Grouped<T, O>& p = *of;
        if constexpr (WAY == Way::ByWeights) return p.m - i0 < BM ? p.m - i0 : BM;
        return rows;
    }
    // goes on from `turn` to the next tile to be summed; the zeros on the way are written
    __device__ __forceinline__ bool next() {
        const Grouped<T, O>& p = *of;
        for (; turn < tiles; turn += gridDim.x) {
            const int what = __builtin_amdgcn_readfirstlane(look());
            // (looked up or not, all lanes have the same: addresses formed of it are scalar)
            row0 = __builtin_amdgcn_readfirstlane(row0), rows = __builtin_amdgcn_readfirstlane(rows);
            kind = __builtin_amdgcn_readfirstlane(kind), slot = __builtin_amdgcn_readfirstlane(slot);
            if (what == 1) return true;
            if (what == 0) continue;
            const int high = out_rows();
            for (int e = threadIdx.x; e < high * (BN / 4); e += blockDim.x)
                if (const int j = j0 + e % (BN / 4) * 4; j < p.n)
                    store_outputs(out_row(e / (BN / 4)), j, p.n, acc4{0.0f, 0.0f, 0.0f, 0.0f});
        }
        return false;
    }
};

// The sums of a workgroup's waves to their rows; `room`: LDS that no one reads any more, for outputs of two bytes.
template <class T, class O, Way WAY, int BM, int BN, int MF, int NF, class W>
__device__ __forceinline__ void put_tile(const W& w, const acc4 (&acc)[MF][NF], int wm, int wn, int lane, std::uint8_t* room) {
    const Grouped<T, O>& p = *w.of;
    const int high = w.out_rows();
    if constexpr (WAY == Way::ByWeights) {
        if (w.slot >= 0) {
#pragma unroll
            for (int f = 0; f < MF; ++f) {
                const int i = wm + 16 * f + lane % 16;
                if (i >= high) continue;
                float* const row = p.partial + (static_cast<i64>(w.slot) * p.m + w.i0 + i) * p.n;
#pragma unroll
                for (int g = 0; g < NF; ++g) store_outputs(row, w.j0 + wn + 16 * g + 4 * (lane / 16), p.n, acc[f][g]);
            }
            return;
        }
    }
    if constexpr (sizeof(O) == 4) {
#pragma unroll
        for (int f = 0; f < MF; ++f) {
            const int i = wm + 16 * f + lane % 16;
            if (i >= high) continue;
            O* const row = w.out_row(i);
#pragma unroll
            for (int g = 0; g < NF; ++g) store_outputs(row, w.j0 + wn + 16 * g + 4 * (lane / 16), p.n, acc[f][g]);
        }
    } else {
        // Values of two bytes are put together in LDS, 16 rows at a time, so that a store is of sixteen bytes a lane and whole lines.
        constexpr int kRow = 16 * NF * 2 + 16, kLanes = NF * 2;
        room += threadIdx.x / 64 * 16 * kRow;
#pragma unroll
        for (int f = 0; f < MF; ++f) {
#pragma unroll
            for (int g = 0; g < NF; ++g) {
                Pack<O, 4> o;
#pragma unroll
                for (int q = 0; q < 4; ++q) o.v[q] = static_cast<O>(acc[f][g][q]);
                __builtin_memcpy(__builtin_assume_aligned(room + lane % 16 * kRow + (16 * g + 4 * (lane / 16)) * 2, 8), &o, 8);
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
            for (int q = 0; q < kLanes / 4; ++q) {
                const int r = lane / kLanes + 64 / kLanes * q, c = lane % kLanes, i = wm + 16 * f + r, j = w.j0 + wn + c * 8;
                const i32x4 v = *reinterpret_cast<const i32x4*>(room + r * kRow + 16 * c);
                if (i < high && j < p.n) store_piece(w.out_row(i), j, p.n, v);
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        }
    }
}

// Rows of 16-bit values that go to LDS by themselves: BM x BN outputs a workgroup, in steps of 64 values of the summed axis.  While one is
// multiplied, the one after it arrives, over the tile's end into the next tile.
//
// 8192 cubed bf16 in 829 us, 1,327 TFLOP/s (a library's product 1,197), the matrix pipe busy 65% of it: a tile of 256 has 2,050
// cycles of matrix instructions a step and as many of LDS (192 KB of fragments, 64 KB that arrive), which overlap as far as each
// fragment is read one ahead of its use.  Steps of 32 with up to five places in LDS, asked for two to four ahead, were slower
// everywhere (2,048 x 2,048 x 2,048 of two types: 39.4 and 33.9 us): it is not the memory's latency that is waited for.
template <class T, class O, Way WAY, int BM, int BN, int WM, int WN>
__global__ void __launch_bounds__(64 * WM * WN, BM + BN > 256 ? 1 : BM + BN > 128 ? 2 : 4) k_grouped_tiles(Grouped<T, O> p) {
    static_assert(sizeof(T) == 2);
    constexpr Lie LA = WAY == Way::ByWeights ? Lie::Columns : Lie::Rows, LB = WAY == Way::Forward ? Lie::Rows : Lie::Columns;
    constexpr int V = 64;
    using A = Step<LA, BM, V>;
    using B = Step<LB, BN, V>;
    constexpr int WAVES = WM * WN, NA = A::kPieces / 64 / WAVES, NB = B::kPieces / 64 / WAVES, MF = BM / WM / 16, NF = BN / WN / 16,
                  Q = V / 32;
    constexpr unsigned kStage = A::kBytes + B::kBytes;
    static_assert(WAVES * 16 * (16 * NF * 2 + 16) <= kStage && (WAY != Way::ByWeights || BM == BN));
    __shared__ __attribute__((aligned(1024))) std::uint8_t lds[2 * kStage];
    const unsigned lds0 = static_cast<unsigned>(reinterpret_cast<std::uintptr_t>((__attribute__((address_space(3))) std::uint8_t*)lds));
    const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const int wm = wave / WN * (BM / WM), wn = wave % WN * (BN / WN);
    using Walker = Walk<T, O, WAY, BM, BN>;
    Walker walk(p);  // the tile that steps are asked for of

    // (the lane's number anew where it is used once a tile: addresses formed of it are not kept across the steps)
    const auto piece = [&](int q) __attribute__((always_inline)) {
        int l = lane;
        asm volatile("" : "+v"(l));
        return (wave + WAVES * q) * 64 + l;
    };
    const T *at_a[NA], *at_b[NB];  // the lane's pieces of the step to come
    int column_a[NA], column_b[NB];  // gathered Columns: the pieces' columns
    // The rows of a's pieces: of gathered Rows of a tile, of gathered Columns of the next step.  The latter are a few for each fetch of a wave,
    // so they are read as scalars, a step ahead: a lane's own reads would be waited for with the step's (8192 cubed by W: 1,409 us, 1,055
    // so).
    constexpr int kIds = 64 / A::kRowPieces;
    using Scalars = const __attribute__((address_space(4))) int*;
    const Scalars scalars = (Scalars)(reinterpret_cast<std::uintptr_t>(walk.order));
    int id[NA];
    struct Asked {
        int v[NA][kIds];
    };
    int values = 0;  // of the summed axis, left
    int absent = 0;  // rows of the tile: from here on none are multiplied, nor read
    const auto ask = [&](int from) __attribute__((always_inline)) {
        Asked to;
#pragma unroll
        for (int q = 0; q < NA; ++q)
#pragma unroll
            for (int i = 0; i < kIds; ++i) {
                const int r = from + (wave + WAVES * q) * kIds + i;
                to.v[q][i] = scalars[walk.row0 + (r < walk.rows ? r : walk.rows - 1)];
            }
        return to;
    };
    const auto pick = [&](const Asked& of) __attribute__((always_inline)) {
#pragma unroll
        for (int q = 0; q < NA; ++q) {
            id[q] = of.v[q][0];
#pragma unroll
            for (int i = 1; i < kIds; ++i) id[q] = lane / A::kRowPieces == i ? of.v[q][i] : id[q];
        }
    };
    // to the first step of the walk's tile
    const auto begin = [&]() __attribute__((always_inline)) {
        if constexpr (WAY == Way::ByWeights) {
            pick(ask(0));
        } else {
#pragma unroll
            for (int q = 0; q < NA; ++q) {
                const int r = A::row_at(piece(q));
                id[q] = walk.order[walk.row0 + (r < walk.rows ? r : walk.rows - 1)];
            }
        }
        if constexpr (WAY == Way::ByWeights) {
            values = walk.rows;
            // (columns past the row's end are no one's: any place of the row does)
#pragma unroll
            for (int q = 0; q < NA; ++q) {
                const int c = walk.i0 + A::piece_at(piece(q)) * 8;
                column_a[q] = c < p.m ? c : 0;
            }
#pragma unroll
            for (int q = 0; q < NB; ++q) {
                const int c = walk.j0 + B::piece_at(piece(q)) * 8;
                column_b[q] = c < p.n ? c : 0;
            }
        } else {
            values = p.k, absent = __builtin_amdgcn_readfirstlane((walk.rows + 15) / 16 * 16);
#pragma unroll
            for (int q = 0; q < NA; ++q) at_a[q] = p.a + id[q] * p.a_stride + A::piece_at(piece(q)) * 8;
            const T* const w = p.b + walk.kind * p.b_kind;
#pragma unroll
            for (int q = 0; q < NB; ++q) {
                const int r = B::row_at(piece(q)), c = B::piece_at(piece(q)) * 8;
                if constexpr (LB == Lie::Rows)
                    at_b[q] = w + (walk.j0 + r < p.n ? walk.j0 + r : p.n - 1) * p.b_stride + c;
                else
                    at_b[q] = w + r * p.b_stride + (walk.j0 + c < p.n ? walk.j0 + c : 0);
            }
        }
    };
    // asks for the step to come, and goes on
    const auto stage = [&](int slot) __attribute__((always_inline)) {
        const unsigned to = __builtin_amdgcn_readfirstlane(lds0 + slot * kStage + wave * 1024);
        const auto all = [&](auto whole) __attribute__((always_inline)) {
            constexpr bool WHOLE = decltype(whole)::value;
            each_of<NA>([&](auto n) __attribute__((always_inline)) {
                constexpr int q = decltype(n)::value;
                const T* at = WAY == Way::ByWeights ? p.a + (id[q] * p.a_stride + column_a[q]) : at_a[q];
                if (!WHOLE) {
                    const int v = LA == Lie::Rows ? A::piece_at(piece(q)) * 8 : A::row_at(piece(q));
                    at = v < values ? at : reinterpret_cast<const T*>(kNothing);
                }
                if (LA == Lie::Rows && (wave + WAVES * q) * kIds >= absent) at = reinterpret_cast<const T*>(kNothing);
                fetch<WAVES * q * 1024>(at, to);
            });
            each_of<NB>([&](auto n) __attribute__((always_inline)) {
                constexpr int q = decltype(n)::value;
                const T* at = WAY == Way::ByWeights ? p.b + (id[q] * p.b_stride + column_b[q]) : at_b[q];
                if (!WHOLE) {
                    const int v = LB == Lie::Rows ? B::piece_at(piece(q)) * 8 : B::row_at(piece(q));
                    at = v < values ? at : reinterpret_cast<const T*>(kNothing);
                }
                fetch<A::kBytes + WAVES * q * 1024>(at, to);
            });
        };
        if (values >= V) all(std::true_type{});
        else all(std::false_type{});
        values -= V;
        if constexpr (WAY != Way::ByWeights) {
#pragma unroll
            for (int q = 0; q < NA; ++q) at_a[q] += V;
#pragma unroll
            for (int q = 0; q < NB; ++q) at_b[q] += LB == Lie::Rows ? static_cast<i64>(V) : V * p.b_stride;
        }
    };

    int slot = 0;
    bool other = false, more = true;  // the walk is a tile ahead of the products; it has not ended
    // asks for one more step, of the walk's tile or the first of the one after
    const auto ahead = [&](int to) __attribute__((always_inline)) {
        if (values <= 0) {
            if (!more) return;
            walk.turn += gridDim.x;
            more = walk.next();
            if (!more) return;
            other = true;
            begin();
        }
        stage(to);
    };
    // by W: the rows of the step that is asked for next
    const auto ask_next = [&]() __attribute__((always_inline)) { return ask(walk.rows - values); };

    if (!walk.next()) return;
    Walker now = walk;  // the tile that is multiplied
    begin();
    stage(0);
    if constexpr (WAY == Way::ByWeights)
        if (values > 0) pick(ask_next());
    for (;;) {
        const int steps = ((WAY == Way::ByWeights ? now.rows : p.k) + V - 1) / V, high = __builtin_amdgcn_readfirstlane(now.out_rows());
        acc4 acc[MF][NF];
#pragma unroll
        for (int f = 0; f < MF; ++f)
#pragma unroll
            for (int g = 0; g < NF; ++g) acc[f][g] = acc4{0.0f, 0.0f, 0.0f, 0.0f};
        const auto sum = [&](auto full) __attribute__((always_inline)) {
            for (int s = 0; s < steps; ++s) {
                arrived();
                __syncthreads();  // the step is there, and all have read the one before
                const std::uint8_t* const tile = lds + slot * kStage;
                slot ^= 1;
                const auto read_a = [&](int f, int q) __attribute__((always_inline)) { return A::read(tile, wm + 16 * f, q, lane); };
                const auto read_b = [&](int g, int q) __attribute__((always_inline)) { return B::read(tile + A::kBytes, wn + 16 * g, q, lane); };
                i32x4 vb[NF], va = read_a(0, 0);
#pragma unroll
                for (int g = 0; g < NF; ++g) vb[g] = read_b(g, 0);
                ahead(slot);
                Asked asked;
#pragma unroll
                for (int q = 0; q < Q; ++q) {
                    if constexpr (WAY == Way::ByWeights)
                        if (q + 1 == Q && values > 0) asked = ask_next();
                    // each fragment is read while the one before is multiplied
                    i32x4 next_b[NF];
#pragma unroll
                    for (int f = 0; f < MF; ++f) {
                        if (!decltype(full)::value && wm + 16 * f >= high) continue;  // no rows of the tile
                        const i32x4 now_a = va;
                        if (f + 1 < MF) va = read_a(f + 1, q);
                        else if (q + 1 < Q) va = read_a(0, q + 1);
                        if (f + 2 == MF && q + 1 < Q)
#pragma unroll
                            for (int g = 0; g < NF; ++g) next_b[g] = read_b(g, q + 1);
#pragma unroll
                        for (int g = 0; g < NF; ++g) acc[f][g] = Multiply<T>::add(vb[g], now_a, acc[f][g]);
                        if (decltype(full)::value) {
                            // (in this order: left to itself the compiler has each read waited for at once)
                            constexpr int kReadsA = LA == Lie::Rows ? 1 : 2, kReadsB = LB == Lie::Rows ? 1 : 2;
                            if (f + 1 < MF || q + 1 < Q) __builtin_amdgcn_sched_group_barrier(0x100, kReadsA, 0);
                            if (f + 2 == MF && q + 1 < Q) __builtin_amdgcn_sched_group_barrier(0x100, kReadsB * NF, 0);
                            __builtin_amdgcn_sched_group_barrier(0x008, NF, 0);
                        }
                    }
                    if (q + 1 < Q) {
                        if (!decltype(full)::value) {
                            va = read_a(0, q + 1);
#pragma unroll
                            for (int g = 0; g < NF; ++g) next_b[g] = read_b(g, q + 1);
                        }
#pragma unroll
                        for (int g = 0; g < NF; ++g) vb[g] = next_b[g];
                    }
                }
                if constexpr (WAY == Way::ByWeights)
                    if (values > 0) pick(asked);
            }
        };
        // (In tiles of 256 a loop each for waves whose fragments all have rows and for others: between conditions the reads would not be
        // ahead.  In smaller ones, whose kernels are short, twice the instructions cost more than the products of no rows: 4,096 rows of
        // 32 types, 1,024 squared, 19.9 us, 21.6 with both.)
        if (WAY == Way::ByWeights || BM < 256 || wm + 16 * MF <= high) sum(std::true_type{});
        else sum(std::false_type{});
        settle_products();
        if constexpr (sizeof(O) == 2) __syncthreads();  // all have read the last step, whose place is used
        put_tile<T, O, WAY, BM, BN, MF, NF>(now, acc, wm, wn, lane, lds + (slot ^ 1) * kStage);
        if (!other) return;  // (a tile's last step has asked for one of the next, if there is one)
        now = walk;
        other = false;
    }
}

// Rows at any alignment, and FP32 ones, which become three bf16 parts on the way: through registers, where a step waits while the one
// before is multiplied.  Steps are of 64 16-bit or 32 FP32 values; one place in LDS, so that several workgroups share a unit and
// one brings a step to LDS while another multiplies.
//
// FP32: x = x1 + x2 + x3 in bf16, each the rest's nearest, and the six products of parts whose orders of size add up to four at most;
// what is left out is below 2^-24 of |x||w|.  8,192 x 4,096 x 4,096 in 1,393 us, 197 TFLOP/s (a library's FP32 product 153): the
// matrix pipe is busy 53% of it, the rest goes to the parts (3.7 vector instructions for each matrix one) and to the one place in LDS.
// Forming the parts between the last products of the step before took 1,500 us; three workgroups a unit spill (2,344).
template <class T, class O, Way WAY, bool ALIGNED, int BM, int BN, int WM, int WN>
__global__ void __launch_bounds__(64 * WM * WN, BM == 128 ? 2 : 4) k_grouped_held(Grouped<T, O> p) {
    constexpr Lie LA = WAY == Way::ByWeights ? Lie::Columns : Lie::Rows, LB = WAY == Way::Forward ? Lie::Rows : Lie::Columns;
    constexpr bool SPLIT = sizeof(T) == 4;
    constexpr int kValues = SPLIT ? 32 : 64, PARTS = SPLIT ? 3 : 1, kPer = 16 / static_cast<int>(sizeof(T));
    using A = Step<LA, BM, kValues>;
    using B = Step<LB, BN, kValues>;
    constexpr int THREADS = 64 * WM * WN, NA = BM * kValues / kPer / THREADS, NB = BN * kValues / kPer / THREADS, MF = BM / WM / 16,
                  NF = BN / WN / 16;
    static_assert(sizeof(O) == 4 || WM * WN * 16 * (16 * NF * 2 + 16) <= (A::kBytes + B::kBytes) * PARTS);
    static_assert(WAY != Way::ByWeights || BM == BN);
    __shared__ __attribute__((aligned(1024))) std::uint8_t lds[(A::kBytes + B::kBytes) * PARTS];
    const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const int wm = wave / WN * (BM / WM), wn = wave % WN * (BN / WN);
    using Walker = Walk<T, O, WAY, BM, BN>;
    Walker walk(p);

    // piece q of the lane: sixteen bytes of the memory's rows, side by side for neighbouring lanes
    const auto row_of = [&](int q, auto rows, int width) {  // width: outer indices
        return (q * THREADS + static_cast<int>(threadIdx.x)) / (decltype(rows)::value ? kValues / kPer : width / kPer);
    };
    const auto column_of = [&](int q, auto rows, int width) {
        return (q * THREADS + static_cast<int>(threadIdx.x)) % (decltype(rows)::value ? kValues / kPer : width / kPer) * kPer;
    };
    constexpr std::bool_constant<LA == Lie::Rows> rows_a{};
    constexpr std::bool_constant<LB == Lie::Rows> rows_b{};
    const T *at_a[NA], *at_b[NB];  // the rows of the lane's pieces; ALIGNED: the pieces of the step to come
    int values = 0, done = 0;  // of the summed axis: left, behind
    const auto begin = [&] {
        values = WAY == Way::ByWeights ? walk.rows : p.k, done = 0;
        if constexpr (WAY != Way::ByWeights) {
#pragma unroll
            for (int q = 0; q < NA; ++q) {
                const int r = row_of(q, rows_a, BM);
                at_a[q] = p.a + walk.order[walk.row0 + (r < walk.rows ? r : walk.rows - 1)] * p.a_stride;
                if constexpr (ALIGNED) at_a[q] += column_of(q, rows_a, BM);
            }
            const T* const w = p.b + walk.kind * p.b_kind;
#pragma unroll
            for (int q = 0; q < NB; ++q) {
                const int r = row_of(q, rows_b, BN), c = column_of(q, rows_b, BN);
                if constexpr (LB == Lie::Rows) {
                    at_b[q] = w + (walk.j0 + r < p.n ? walk.j0 + r : p.n - 1) * p.b_stride;
                    if constexpr (ALIGNED) at_b[q] += c;
                } else {
                    at_b[q] = w + r * p.b_stride;
                    if constexpr (ALIGNED) at_b[q] += walk.j0 + c < p.n ? walk.j0 + c : 0;
                }
            }
        }
    };
    i32x4 held_a[NA], held_b[NB];
    int id[NA];  // gathered Columns: the rows of the step to come
    const auto ask = [&] {
        if constexpr (WAY == Way::ByWeights)
#pragma unroll
            for (int q = 0; q < NA; ++q) {
                const int r = row_of(q, rows_a, BM);
                id[q] = walk.order[walk.row0 + done + (r < values ? r : values - 1)];
            }
    };
    // column and row's end of a's and b's pieces of the step `at` values on
    const auto columns_a = [&](int q, int at) {
        return LA == Lie::Rows ? at + column_of(q, rows_a, BM) : walk.i0 + column_of(q, rows_a, BM);
    };
    const auto columns_b = [&](int q, int at) {
        return LB == Lie::Rows ? at + column_of(q, rows_b, BN) : walk.j0 + column_of(q, rows_b, BN);
    };
    const int end_a = WAY == Way::ByWeights ? p.m : p.k, end_b = WAY == Way::Forward ? p.k : p.n;
    // asks for the step to come, and goes on; pieces that pass a row's end are settled when they are used
    const auto load = [&] {
        if constexpr (ALIGNED) {
            const auto all = [&](auto whole) {
                constexpr bool WHOLE = decltype(whole)::value;
                const auto from = [&](const T* at, int v) {
                    return load_sixteen(WHOLE || v < values ? static_cast<const void*>(at) : kNothing);
                };
#pragma unroll
                for (int q = 0; q < NA; ++q) {
                    const int r = row_of(q, rows_a, BM), c = column_of(q, rows_a, BM);
                    if constexpr (LA == Lie::Rows) held_a[q] = from(at_a[q], c);
                    else held_a[q] = from(p.a + id[q] * p.a_stride + (walk.i0 + c < p.m ? walk.i0 + c : 0), r);
                }
#pragma unroll
                for (int q = 0; q < NB; ++q) {
                    const int r = row_of(q, rows_b, BN), c = column_of(q, rows_b, BN);
                    if constexpr (LB == Lie::Rows) held_b[q] = from(at_b[q], c);
                    else if constexpr (WAY == Way::ByRows) held_b[q] = from(at_b[q], r);
                    else held_b[q] = from(p.b + id[q] * p.b_stride + (walk.j0 + c < p.n ? walk.j0 + c : 0), r);
                }
            };
            if (values >= kValues) all(std::true_type{});
            else all(std::false_type{});
            if constexpr (WAY != Way::ByWeights) {
#pragma unroll
                for (int q = 0; q < NA; ++q) at_a[q] += kValues;
#pragma unroll
                for (int q = 0; q < NB; ++q) at_b[q] += LB == Lie::Rows ? static_cast<i64>(kValues) : kValues * p.b_stride;
            }
        } else {
#pragma unroll
            for (int q = 0; q < NA; ++q) {
                const T* row;
                if constexpr (LA == Lie::Rows) row = at_a[q];
                else row = row_of(q, rows_a, BM) < values ? p.a + id[q] * p.a_stride : nullptr;
                held_a[q] = row ? load_piece(row, columns_a(q, done), end_a) : i32x4{0, 0, 0, 0};
            }
#pragma unroll
            for (int q = 0; q < NB; ++q) {
                const T* row;
                if constexpr (LB == Lie::Rows) row = at_b[q];
                else if constexpr (WAY == Way::ByRows) row = row_of(q, rows_b, BN) < values ? at_b[q] + done * p.b_stride : nullptr;
                else row = row_of(q, rows_b, BN) < values ? p.b + id[q] * p.b_stride : nullptr;
                held_b[q] = row ? load_piece(row, columns_b(q, done), end_b) : i32x4{0, 0, 0, 0};
            }
        }
        values -= kValues, done += kValues;
        if (values > 0) ask();
    };
    const auto settled = [&](i32x4 w, int c, int end) {
        if constexpr (ALIGNED) return w;
        else return settle_piece<T>(w, c, end);
    };
    const auto put = [&](auto step, std::uint8_t* to, int row, int column, i32x4 w) {
        using S = decltype(step);
        if constexpr (SPLIT) {
            const FourParts f = split_four(w);
#pragma unroll
            for (int k = 0; k < 3; ++k)
                *reinterpret_cast<uint2*>(to + k * S::kBytes + S::place(row, column / 8, column / 4 % 2)) = f.part[k];
        } else {
            *reinterpret_cast<i32x4*>(to + S::place(row, column / 8, 0)) = w;
        }
    };

    bool more = walk.next();
    if (!more) return;
    begin();
    ask();
    load();
    while (more) {
        const Walker now = walk;
        const int steps = ((WAY == Way::ByWeights ? now.rows : p.k) + kValues - 1) / kValues, high = __builtin_amdgcn_readfirstlane(now.out_rows());
        acc4 acc[MF][NF];
#pragma unroll
        for (int f = 0; f < MF; ++f)
#pragma unroll
            for (int g = 0; g < NF; ++g) acc[f][g] = acc4{0.0f, 0.0f, 0.0f, 0.0f};
        for (int s = 0; s < steps; ++s) {
            __syncthreads();  // all have read the step before
#pragma unroll
            for (int q = 0; q < NA; ++q)
                put(A{}, lds, row_of(q, rows_a, BM), column_of(q, rows_a, BM),
                    settled(held_a[q], columns_a(q, done - kValues), end_a));
#pragma unroll
            for (int q = 0; q < NB; ++q)
                put(B{}, lds + A::kBytes * PARTS, row_of(q, rows_b, BN), column_of(q, rows_b, BN),
                    settled(held_b[q], columns_b(q, done - kValues), end_b));
            __syncthreads();
            if (s + 1 == steps) {
                walk.turn += gridDim.x;
                more = walk.next();
                if (more) begin(), ask();
            }
            if (more) load();
            if constexpr (SPLIT) {
                // two columns of fragments at a time, so that the registers are those of two workgroups a unit
                constexpr int kAtOnce = NF < 2 ? NF : 2;
#pragma unroll
                for (int g0 = 0; g0 < NF; g0 += kAtOnce) {
                    Parts vb[kAtOnce];
#pragma unroll
                    for (int g = 0; g < kAtOnce; ++g)
#pragma unroll
                        for (int k = 0; k < 3; ++k)
                            vb[g].part[k] = B::read(lds + A::kBytes * PARTS + k * B::kBytes, wn + 16 * (g0 + g), 0, lane);
                    Parts va;
#pragma unroll
                    for (int k = 0; k < 3; ++k) va.part[k] = A::read(lds + k * A::kBytes, wm, 0, lane);
#pragma unroll
                    for (int f = 0; f < MF; ++f) {
                        if (wm + 16 * f >= high) break;
                        const Parts now_a = va;
                        if (f + 1 < MF)
#pragma unroll
                            for (int k = 0; k < 3; ++k) va.part[k] = A::read(lds + k * A::kBytes, wm + 16 * (f + 1), 0, lane);
#pragma unroll
                        for (int g = 0; g < kAtOnce; ++g) acc[f][g0 + g] = add_parts(vb[g], now_a, acc[f][g0 + g]);
                    }
                }
            } else {
                i32x4 vb[NF][2];
#pragma unroll
                for (int g = 0; g < NF; ++g)
#pragma unroll
                    for (int q = 0; q < 2; ++q) vb[g][q] = B::read(lds + A::kBytes, wn + 16 * g, q, lane);
#pragma unroll
                for (int f = 0; f < MF; ++f)
#pragma unroll
                    for (int q = 0; q < 2; ++q) {
                        if (wm + 16 * f >= high) break;
                        const i32x4 va = A::read(lds, wm + 16 * f, q, lane);
#pragma unroll
                        for (int g = 0; g < NF; ++g) acc[f][g] = Multiply<T>::add(vb[g][q], va, acc[f][g]);
                    }
            }
        }
        settle_products();
        if constexpr (sizeof(O) == 2) __syncthreads();  // all have read the last step, whose place is used
        put_tile<T, O, WAY, BM, BN, MF, NF>(now, acc, wm, wn, lane, lds);
    }
}

// The sums of kinds whose rows are cut: rows of workgroups take these kinds in turn and join their runs in order, four neighbouring
// values a lane.  Bytes of the parts bound it: 59 runs of 256 x 512 (31 MB) in 9.9 us.
template <class O>
__global__ void __launch_bounds__(256) k_grouped_join(Grouped<O, O> p) {
    const int kinds = p.kinds, lane = threadIdx.x % 64;
    if (!plan_fits(p.plan, p.tokens, kinds)) return;
    const int run = run_of(p.plan, p.tokens, p.round, p.least);
    if (run > p.tokens) return;
    const int* const offsets = p.plan + plan_offsets();
    const i64 size = static_cast<i64>(p.m) * p.n;
    unsigned nth = 0;
    for (int base = 0; base < kinds; base += 64) {
        const int mine = base + lane < kinds ? base + lane : kinds - 1, from = offsets[mine], to = offsets[mine + 1];
        unsigned long long cut = __ballot(base + lane < kinds && to > from && from / run != (to - 1) / run);
        for (; cut; cut &= cut - 1) {
            if (nth++ % gridDim.y != blockIdx.y) continue;
            const int at = __builtin_ctzll(cut), kind = base + at;
            const int first = __builtin_amdgcn_readlane(from, at) / run, last = (__builtin_amdgcn_readlane(to, at) - 1) / run;
            for (i64 e = 4 * (static_cast<i64>(blockIdx.x) * 256 + threadIdx.x); e < size; e += 1024LL * gridDim.x) {
                const auto part = [&](int slot) {
                    const float* const at = p.partial + slot * size + e;
                    if (e + 4 <= size) return *reinterpret_cast<const Pack<float, 4>*>(at);
                    Pack<float, 4> v;
#pragma unroll
                    for (int q = 0; q < 4; ++q) v.v[q] = e + q < size ? at[q] : 0.0f;
                    return v;
                };
                Pack<float, 4> sum = part(2 * first + 1);
#pragma unroll 8
                for (int r = first + 1; r <= last; ++r) {
                    const Pack<float, 4> v = part(2 * r);
#pragma unroll
                    for (int q = 0; q < 4; ++q) sum.v[q] += v.v[q];
                }
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    if (e + q < size)
                        p.out[kind * p.out_kind + (e + q) / p.n * p.out_stride + (e + q) % p.n] = static_cast<O>(sum.v[q]);
            }
        }
    }
}

// Up to 16 rows of a kind: 16 NF outputs a workgroup, which reads their weights once for its rows; a kind of more rows has them
// read, from the caches mostly, for each 16.  KS waves share the summed axis.  The weights' bytes bound it: one row, 2,048 x 4,096
// of bf16, 5.8 us (2.9 TB/s, the launch among it); 147 rows of 32 kinds, 1,024 x 2,048 of f16 (134 MB, partly in the last cache),
// 22.6 us, 5.9 TB/s.
template <class T, class O, bool DIRECT, int NF, int KS>
__global__ void __launch_bounds__(64 * KS) k_grouped_rows(Grouped<T, O> p) {
    __shared__ FewRoom<T, NF, KS> room;
    const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const int present = p.plan[0], u = blockIdx.x / p.tiles_n, j0 = blockIdx.x % p.tiles_n * 16 * NF;
    if (u >= present + p.tokens / 16 || !plan_fits(p.plan, p.tokens, p.kinds)) return;
    const int* const start = p.plan + plan_start(p.kinds);
    const int* const order = p.plan + plan_order(p.kinds);
    const int at = last_up_to(u, present, [&](int q) { return q + start[q] / 16; });
    const int row0 = start[at] + (u - at - start[at] / 16) * 16, kind = p.plan[plan_present(p.kinds) + at];
    const int rows = start[at + 1] - row0 < 16 ? start[at + 1] - row0 : 16, row = lane % 16;
    if (rows <= 0) return;
    const int id = order[row0 + (row < rows ? row : rows - 1)];
    if (kind < p.kinds) {
        const T* b[NF];
#pragma unroll
        for (int g = 0; g < NF; ++g) {
            const int j = j0 + 16 * g + row;
            b[g] = p.b + kind * p.b_kind + (j < p.n ? j : p.n - 1) * p.b_stride;
        }
        few_rows<T, DIRECT, NF, KS>(p.a + id * p.a_stride, b, p.k, room);
    }
    if (row >= rows) return;
    for (int g = wave; g < NF; g += KS)
        store_outputs(p.out + id * p.out_stride, j0 + 16 * g + 4 * (lane / 16), p.n,
                      kind < p.kinds ? joined(room, g) : acc4{0.0f, 0.0f, 0.0f, 0.0f});
}

// How a call is cut (node_grouped.hip).
struct Cut {
    int tile;  // 256, 128, 64, or 16: k_grouped_rows
    bool direct;  // rows are aligned to 16 bytes, and as long as whole ones
    int units;    // of 16 rows, at most
    int columns, waves;  // of a workgroup of k_grouped_rows: 64 and 2 or 4, or 16 and 4 or 8
};

template <class T, class O>
void launch_grouped(const Grouped<T, O>& p, Way way, const Cut& cut, hipStream_t stream) {
    const auto tiles = [&](auto w) {
        constexpr Way W = decltype(w)::value;
        if constexpr (sizeof(T) == 2) {
            if (cut.direct) {
                switch (cut.tile) {
                    case 256: k_grouped_tiles<T, O, W, 256, 256, 2, 4><<<kComputeUnits, 512, 0, stream>>>(p); break;
                    case 128: k_grouped_tiles<T, O, W, 128, 128, 2, 2><<<2 * kComputeUnits, 256, 0, stream>>>(p); break;
                    default: k_grouped_tiles<T, O, W, 64, 64, 2, 2><<<4 * kComputeUnits, 256, 0, stream>>>(p);
                }
                SMX_LAUNCH_CHECK("k_grouped_tiles");
                return;
            }
        }
        const auto held = [&](auto aligned_rows) {
            constexpr bool ALIGNED = decltype(aligned_rows)::value;
            if (cut.tile == 128)
                k_grouped_held<T, O, W, ALIGNED, 128, 128, 2, 2><<<2 * kComputeUnits, 256, 0, stream>>>(p);
            else
                k_grouped_held<T, O, W, ALIGNED, 64, 64, 2, 2><<<4 * kComputeUnits, 256, 0, stream>>>(p);
        };
        if constexpr (sizeof(T) == 4) {
            if (cut.direct) held(std::true_type{});
            else held(std::false_type{});
        } else {
            held(std::false_type{});
        }
        SMX_LAUNCH_CHECK("k_grouped_held");
    };
    using std::integral_constant;
    if (way == Way::ByRows) return tiles(integral_constant<Way, Way::ByRows>{});
    if (way == Way::ByWeights) return tiles(integral_constant<Way, Way::ByWeights>{});
    if (cut.tile != 16) return tiles(integral_constant<Way, Way::Forward>{});
    const auto rows = [&](auto nf, auto ks) {
        constexpr int NF = decltype(nf)::value, KS = decltype(ks)::value;
        const unsigned grid = static_cast<unsigned>(cut.units) * static_cast<unsigned>(p.tiles_n);
        if (cut.direct)
            k_grouped_rows<T, O, true, NF, KS><<<grid, 64 * KS, 0, stream>>>(p);
        else
            k_grouped_rows<T, O, false, NF, KS><<<grid, 64 * KS, 0, stream>>>(p);
    };
    if (cut.columns == 64 && cut.waves == 2) rows(integral_constant<int, 4>{}, integral_constant<int, 2>{});
    else if (cut.columns == 64) rows(integral_constant<int, 4>{}, integral_constant<int, 4>{});
    else if (cut.waves == 4) rows(integral_constant<int, 1>{}, integral_constant<int, 4>{});
    else rows(integral_constant<int, 1>{}, integral_constant<int, 8>{});
    SMX_LAUNCH_CHECK("k_grouped_rows");
}

}  // namespace node
}  // namespace smx
