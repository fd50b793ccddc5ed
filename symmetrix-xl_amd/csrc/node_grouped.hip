// Products of rows with the weights of their kind, and their gradients: how calls are cut, and the C entries.
#include "node_grouped.hpp"

namespace smx {
namespace node {

extern template void launch_grouped<float, float>(const Grouped<float, float>&, Way, const Cut&, hipStream_t);
extern template void launch_grouped<bf16, float>(const Grouped<bf16, float>&, Way, const Cut&, hipStream_t);
extern template void launch_grouped<bf16, bf16>(const Grouped<bf16, bf16>&, Way, const Cut&, hipStream_t);
extern template void launch_grouped<f16, float>(const Grouped<f16, float>&, Way, const Cut&, hipStream_t);
extern template void launch_grouped<f16, f16>(const Grouped<f16, f16>&, Way, const Cut&, hipStream_t);

namespace {

// f(T{}, O{}): outputs are of the rows' type or FP32
template <class F>
void with_types(int dtype, int out_dtype, F&& f) {
    with_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        if (out_dtype == SMX_DTYPE_F32) return f(T{}, float{});
        if constexpr (sizeof(T) == 2) f(T{}, T{});
    });
}

// What tiles of 256, 128 and 64 cost, in us: a step of 64 values of the summed axis with `filled` tiles on a unit, which holds one,
// two or four of them, and what a tile takes beside its steps (measured: 8192 cubed, and 2,048 rows of 2,048 values).
constexpr int kSizes[3] = {256, 128, 64};
int held(int tile) { return tile == 256 ? 1 : tile == 128 ? 2 : 4; }
double step_time(int tile, i64 filled) {
    if (tile == 256) return 1.9;
    if (tile == 128) return 1.15;
    return 0.5 + 0.19 * static_cast<double>(filled < 4 ? filled : 4);
}
double tile_time(int tile, i64 steps, i64 filled) {
    return static_cast<double>(steps) * step_time(tile, filled) + (tile == 256 ? 4.0 : tile == 128 ? 2.5 : 2.0);
}

i64 ceil_of(i64 a, i64 b) { return (a + b - 1) / b; }

// The tile that takes least by these for `units(tile)` of rows and n columns; tiles through registers are of 128 or 64.
template <class F>
int tile_for(F&& units, i64 n, i64 k, bool largest) {
    int best = 64;
    double least = 1e300;
    for (const int t : kSizes) {
        if (t == 256 && !largest) continue;
        const i64 count = units(t) * ceil_of(n, t), card = held(t) * kComputeUnits;
        const double cost = static_cast<double>(ceil_of(count, card)) * tile_time(t, ceil_of(k, 64), ceil_of(count, kComputeUnits));
        if (cost < least) least = cost, best = t;
    }
    return best;
}

// Rows of a kind, in the mean over the kinds of the table, up to which k_grouped_rows is taken: how many kinds have rows is known to
// the device alone.  Where few have, this is not the faster one (512 x 1,024 bf16: 8,192 rows in 5 of 512 types 82 us, 23 as a
// table of 5, which takes tiles; 1,400 rows in 5 of 89 types 19 and 8; spread over all types the weights bound it, 149 and 27 us).
constexpr i64 kFewRows = 16;

Cut cut_rows(Way way, i64 rows, i64 kinds, i64 n, i64 inner, bool direct, bool split) {
    Cut c{128, direct, 0, 0, 0};
    const i64 k = kinds < rows ? kinds : rows;
    if (way == Way::Forward && rows <= k * kFewRows) {
        // Columns and waves of a workgroup: 64 where that still makes two a unit, and the waves such that each has eight steps or more, of
        // which four are under way (147 rows of 32 types, 1,024 x 2,048: 22.4 us at 64 and 2, 25.7 at 64 and 4, 48.6 at 16 and
        // 8; 64 of 8, 4,096 squared FP32: 162, 114 and 118; one row, 2,048 x 4,096: 10.4, 10.1 and 8.2, 7.7 at 16 and 4).
        const i64 units = (kinds + 1 < rows ? kinds + 1 : rows) + rows / 16, steps = ceil_of(inner * (split ? 4 : 2), kStepBytes);
        c.units = static_cast<int>(units);
        c.columns = units * ceil_of(n, 64) >= 2 * kComputeUnits ? 64 : 16;
        c.waves = (c.columns == 64 ? 2 : 4) * (steps >= 64 ? 2 : 1);
        // (a launch has fewer than 2^32 threads; the tiles' are as many as the card holds)
        if (units * ceil_of(n, c.columns) * 64 * c.waves < (1LL << 32)) {
            c.tile = 16;
            return c;
        }
    }
    // (rows spread evenly over the kinds: their numbers are known to the device alone)
    c.tile = tile_for([&](i64 t) { return k * ceil_of(ceil_of(rows, k), t); }, n, inner, direct && !split);
    return c;
}

// The weights' gradient of m x n a kind: the tile, the units of rows that the card holds at once, and the least run, so that no more
// than two rounds are cut (run_of): 0 where none can be.
struct Runs {
    int tile;
    i64 round, least, slots;
};

Runs runs_for(i64 rows, i64 kinds, i64 m, i64 n, bool largest) {
    Runs best{};
    double least = 1e300;
    const i64 k = kinds < rows ? kinds : rows < 1 ? 1 : rows, each = ceil_of(rows < 1 ? 1 : rows, k);
    for (const int t : kSizes) {
        if (t == 256 && !largest) continue;
        const i64 per = ceil_of(m, t) * ceil_of(n, t), card = held(t) * kComputeUnits, round = per < card ? card / per : 1;
        i64 run = ceil_of(rows, 2 * round);
        run = run < 512 ? 512 : ceil_of(run, 64) * 64;
        // (rows spread evenly: cut into two rounds at most, or not)
        const auto cost_of = [&](i64 rounds, i64 r) {
            return static_cast<double>(rounds) * tile_time(t, ceil_of(r, 64), ceil_of(k * per, kComputeUnits));
        };
        double cost = cost_of(ceil_of(k * per, card), each);
        if (round > k) {
            const i64 cut = ceil_of(rows, round - k) < run ? run : ceil_of(rows, round - k);
            if (const double c = cost_of(1, cut) + 10; cut < each && c < cost) cost = c;
        }
        if (cost < least) {
            least = cost;
            // (where a type's tiles fill the card, run_of cuts none: two rounds less one type are no more than one unit)
            const bool cut = round > 1 && run < rows;
            best = {t, round, cut ? run : 0, cut ? 2 * (rows / run + 1) : 0};
        }
    }
    return best;
}

bool wide(const void* p, i64 stride, i64 cols, int size) {
    return aligned(p, 16) && stride * size % 16 == 0 && cols * size % 16 == 0;
}

void check_kinds(i64 rows, i64 kinds) {
    require(rows >= 0 && rows <= (1LL << 30), "rows must be in [0, 2^30]");
    require(kinds >= 1, "there must be a kind at least");
    if (kinds > kMostKinds) throw std::domain_error("products by kind take up to 4096 kinds");
}

bool widths_ok(i64 a, i64 b) { return a <= (1 << 24) && b <= (1 << 24); }

void check_width(i64 v, const char* what) {
    if (v < 0 || v > (1 << 24)) throw std::invalid_argument(std::string(what) + " must be in [0, 2^24]");
}

void check_weights(const void* w, i64 stride, i64 kind_stride, i64 kinds, i64 rows, i64 cols, int dtype, const char* name) {
    check_rows(w, stride, rows, cols, dtype, name);
    if (kinds > 1 && rows > 0 && cols > 0 && kind_stride < (rows - 1) * (rows > 1 ? stride : 0) + cols)
        throw std::invalid_argument(std::string(name) + ": the matrices of two kinds overlap");
}

void check_plan(const void* plan) { require(plan && aligned(plan, 16), "the plan is NULL or not 16-byte aligned"); }

void check_types(int dtype, int out_dtype) {
    require(dtype >= SMX_DTYPE_F32 && dtype <= SMX_DTYPE_F16, "unknown dtype code");
    require(out_dtype == dtype || out_dtype == SMX_DTYPE_F32, "products by kind are of the rows' type or FP32");
}

template <class T, class O>
void product(Way way, const void* a, i64 a_stride, const void* w, i64 w_stride, i64 w_kind, const void* plan, i64 rows, i64 kinds,
             i64 k, i64 n, void* out, i64 out_stride, hipStream_t stream) {
    Grouped<T, O> p{};
    p.a = static_cast<const T*>(a), p.a_stride = a_stride;
    p.b = static_cast<const T*>(w), p.b_stride = w_stride, p.b_kind = w_kind;
    p.out = static_cast<O*>(out), p.out_stride = out_stride;
    p.plan = static_cast<const int*>(plan);
    p.tokens = static_cast<int>(rows), p.kinds = static_cast<int>(kinds);
    p.n = static_cast<int>(n), p.k = static_cast<int>(k);
    const i64 w_cols = way == Way::Forward ? k : n;
    const bool direct = wide(a, a_stride, k, sizeof(T)) && wide(w, w_stride, w_cols, sizeof(T)) &&
                        (kinds == 1 || w_kind * static_cast<i64>(sizeof(T)) % 16 == 0);
    const Cut cut = cut_rows(way, rows, kinds, n, k, direct, sizeof(T) == 4);
    p.tiles_m = 1, p.tiles_n = static_cast<int>(ceil_of(n, cut.tile == 16 ? cut.columns : cut.tile));
    require((kinds + 1 + rows / cut.tile) * p.tiles_n < (1LL << 31), "the product has too many tiles");
    launch_grouped<T, O>(p, way, cut, stream);
}

template <class T, class O>
void weights_gradient(const void* grad, i64 grad_stride, const void* x, i64 x_stride, const void* plan, i64 rows, i64 kinds, i64 m,
                      i64 n, void* out, i64 out_stride, i64 out_kind, void* workspace, hipStream_t stream) {
    Grouped<T, O> p{};
    p.a = static_cast<const T*>(grad), p.a_stride = grad_stride;
    p.b = static_cast<const T*>(x), p.b_stride = x_stride;
    p.out = static_cast<O*>(out), p.out_stride = out_stride, p.out_kind = out_kind;
    p.plan = static_cast<const int*>(plan);
    p.tokens = static_cast<int>(rows), p.kinds = static_cast<int>(kinds);
    p.m = static_cast<int>(m), p.n = static_cast<int>(n);
    const bool direct = wide(grad, grad_stride, m, sizeof(T)) && wide(x, x_stride, n, sizeof(T));
    const Runs runs = runs_for(rows, kinds, m, n, direct && sizeof(T) == 2);
    p.round = static_cast<int>(runs.round), p.least = static_cast<int>(runs.least);
    const Cut cut{runs.tile, direct, 0, 0, 0};
    p.tiles_m = static_cast<int>((m + cut.tile - 1) / cut.tile), p.tiles_n = static_cast<int>((n + cut.tile - 1) / cut.tile);
    require((kinds + (runs.least ? rows / runs.least : 0)) * p.tiles_m * p.tiles_n < (1LL << 31), "the product has too many tiles");
    p.partial = static_cast<float*>(workspace);
    launch_grouped<T, O>(p, Way::ByWeights, cut, stream);
    if (runs.least > 0) {
        Grouped<O, O> j{};
        j.out = p.out, j.out_stride = out_stride, j.out_kind = out_kind;
        j.plan = p.plan, j.tokens = p.tokens, j.kinds = p.kinds, j.m = p.m, j.n = p.n;
        j.round = p.round, j.least = p.least, j.partial = p.partial;
        // (few workgroups: whether there is anything to join is known to the device alone)
        const i64 blocks = ceil_of(m * n, 1024), cuts = (rows - 1) / runs.least, most = kinds < cuts ? kinds : cuts;
        k_grouped_join<O><<<dim3(static_cast<unsigned>(blocks < 256 ? blocks : 256), static_cast<unsigned>(most < 4 ? most : 4)), 256, 0,
                            stream>>>(j);
        SMX_LAUNCH_CHECK("k_grouped_join");
    }
}

}  // namespace
}  // namespace node
}  // namespace smx

using namespace smx;
using namespace smx::node;

extern "C" {

int32_t smx_grouped_linear(const void* x, int64_t x_stride, int32_t dtype, const void* w, int64_t w_stride, int64_t w_type_stride,
                           const void* plan, int64_t rows, int64_t num_types, int64_t inputs, int64_t outputs, int32_t out_dtype,
                           void* out, int64_t out_stride, void* stream) {
    return guarded([&] {
        check_types(dtype, out_dtype);
        check_kinds(rows, num_types);
        check_width(inputs, "inputs"), check_width(outputs, "outputs");
        check_rows(x, x_stride, rows, inputs, dtype, "x");
        check_weights(w, w_stride, w_type_stride, num_types, outputs, inputs, dtype, "w");
        check_rows(out, out_stride, rows, outputs, out_dtype, "out");
        check_plan(plan);
        if (rows == 0 || outputs == 0) return;
        with_types(dtype, out_dtype, [&](auto t, auto o) {
            product<decltype(t), decltype(o)>(Way::Forward, x, x_stride, w, w_stride, w_type_stride, plan, rows, num_types, inputs,
                                              outputs, out, out_stride, static_cast<hipStream_t>(stream));
        });
    });
}

int32_t smx_grouped_linear_by_rows(const void* grad, int64_t grad_stride, int32_t dtype, const void* w, int64_t w_stride,
                                   int64_t w_type_stride, const void* plan, int64_t rows, int64_t num_types, int64_t inputs,
                                   int64_t outputs, int32_t out_dtype, void* dx, int64_t dx_stride, void* stream) {
    return guarded([&] {
        check_types(dtype, out_dtype);
        check_kinds(rows, num_types);
        check_width(inputs, "inputs"), check_width(outputs, "outputs");
        check_rows(grad, grad_stride, rows, outputs, dtype, "grad");
        check_weights(w, w_stride, w_type_stride, num_types, outputs, inputs, dtype, "w");
        check_rows(dx, dx_stride, rows, inputs, out_dtype, "dx");
        check_plan(plan);
        if (rows == 0 || inputs == 0) return;
        with_types(dtype, out_dtype, [&](auto t, auto o) {
            product<decltype(t), decltype(o)>(Way::ByRows, grad, grad_stride, w, w_stride, w_type_stride, plan, rows, num_types,
                                              outputs, inputs, dx, dx_stride, static_cast<hipStream_t>(stream));
        });
    });
}

int64_t smx_grouped_linear_by_weights_workspace(int64_t rows, int64_t num_types, int64_t inputs, int64_t outputs) {
    if (rows <= 0 || num_types <= 0 || inputs <= 0 || outputs <= 0) return 0;
    if (!widths_ok(inputs, outputs)) return 0;
    // (for rows at any alignment)
    const i64 a = runs_for(rows, num_types, outputs, inputs, true).slots, b = runs_for(rows, num_types, outputs, inputs, false).slots;
    return 4 * (a > b ? a : b) * outputs * inputs;
}

int32_t smx_grouped_linear_by_weights(const void* grad, int64_t grad_stride, const void* x, int64_t x_stride, int32_t dtype,
                                      const void* plan, int64_t rows, int64_t num_types, int64_t inputs, int64_t outputs,
                                      int32_t out_dtype, void* dw, int64_t dw_stride, int64_t dw_type_stride, void* workspace,
                                      int64_t workspace_bytes, void* stream) {
    return guarded([&] {
        check_types(dtype, out_dtype);
        check_kinds(rows, num_types);
        check_width(inputs, "inputs"), check_width(outputs, "outputs");
        check_rows(grad, grad_stride, rows, outputs, dtype, "grad");
        check_rows(x, x_stride, rows, inputs, dtype, "x");
        check_weights(dw, dw_stride, dw_type_stride, num_types, outputs, inputs, out_dtype, "dw");
        check_plan(plan);
        check_workspace(workspace, workspace_bytes, smx_grouped_linear_by_weights_workspace(rows, num_types, inputs, outputs));
        if (inputs == 0 || outputs == 0) return;
        with_types(dtype, out_dtype, [&](auto t, auto o) {
            weights_gradient<decltype(t), decltype(o)>(grad, grad_stride, x, x_stride, plan, rows, num_types, outputs, inputs, dw,
                                                       dw_stride, dw_type_stride, workspace, static_cast<hipStream_t>(stream));
        });
    });
}

}  // extern "C"
