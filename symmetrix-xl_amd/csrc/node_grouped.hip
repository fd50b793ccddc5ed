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

// The tile whose rounds over the card take least, for `units` of rows of a tile: a unit holds one tile of 256, two of 128 or four of
// 64.  Tiles through registers are of 128 or 64.
template <class F>
int tile_for(F&& units, i64 n, bool direct) {
    const auto cost = [&](i64 t, i64 held, double work) {
        const i64 count = units(t) * ((n + t - 1) / t);
        return work / static_cast<double>(held) * static_cast<double>((count + held * kComputeUnits - 1) / (held * kComputeUnits));
    };
    const double c256 = cost(256, 1, 1.0), c128 = cost(128, 2, 1.12), c64 = cost(64, 4, 1.86);
    if (direct && c256 <= c128 && c256 <= c64) return 256;
    return c128 <= c64 ? 128 : 64;
}

// Rows of a kind up to which k_grouped_rows reads its weights straight to registers.
constexpr i64 kFewRows = 16;

Cut cut_rows(Way way, i64 rows, i64 kinds, i64 n, bool direct) {
    Cut c{128, direct, 0};
    const i64 k = kinds < rows ? kinds : rows;
    if (way == Way::Forward && rows <= k * kFewRows) {
        const i64 units = (kinds + 1 < rows ? kinds + 1 : rows) + rows / 16;
        if (units * ((n + 15) / 16) < (1LL << 31)) {
            c.tile = 16, c.units = static_cast<int>(units);
            return c;
        }
    }
    // (rows spread evenly over the kinds: their numbers are known to the device alone)
    c.tile = tile_for([&](i64 t) { return k * (((rows + k - 1) / k + t - 1) / t); }, n, direct);
    return c;
}

// Rows summed together in the weights' gradient: as many as leave two tiles of 128 to each unit if one kind had them all.
i64 run_for(i64 rows, i64 m, i64 n) {
    const i64 tiles = (m + 127) / 128 * ((n + 127) / 128);
    i64 run = (rows * tiles / (2 * kComputeUnits) + 255) / 256 * 256;
    if (run < 512) run = 512;
    return run < rows ? run : rows + 1;  // (not cut)
}

i64 cuts_of(i64 rows, i64 run) { return rows > 0 ? (rows - 1) / run : 0; }

bool wide(const void* p, i64 stride, i64 cols, int size) {
    return aligned(p, 16) && stride * size % 16 == 0 && cols * size % 16 == 0;
}

void check_kinds(i64 rows, i64 kinds) {
    require(rows >= 0 && rows <= (1LL << 30), "rows must be in [0, 2^30]");
    require(kinds >= 1, "there must be a kind at least");
    if (kinds > kMostKinds) throw std::domain_error("products by kind take up to 4096 kinds");
}

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
    const bool aligned_rows = wide(a, a_stride, k, sizeof(T)) && wide(w, w_stride, w_cols, sizeof(T)) &&
                              (kinds == 1 || w_kind * static_cast<i64>(sizeof(T)) % 16 == 0);
    const bool direct = sizeof(T) == 2 && aligned_rows;
    Cut cut = cut_rows(way, rows, kinds, n, direct);
    if (cut.tile == 16) cut.direct = aligned_rows;
    p.tiles_m = 1, p.tiles_n = static_cast<int>((n + cut.tile - 1) / cut.tile);
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
    const bool direct = sizeof(T) == 2 && wide(grad, grad_stride, m, sizeof(T)) && wide(x, x_stride, n, sizeof(T));
    const i64 run = run_for(rows, m, n), cuts = cuts_of(rows, run);
    p.run = static_cast<int>(run), p.units = static_cast<int>(kinds + rows / run);
    Cut cut{tile_for([&](i64 t) { return (kinds < rows ? kinds : rows) * ((m + t - 1) / t) + cuts; }, n, direct), direct, 0};
    p.tiles_m = static_cast<int>((m + cut.tile - 1) / cut.tile), p.tiles_n = static_cast<int>((n + cut.tile - 1) / cut.tile);
    require(p.units * static_cast<i64>(p.tiles_m) * p.tiles_n < (1LL << 31), "the product has too many tiles");
    p.partial = static_cast<float*>(workspace);
    launch_grouped<T, O>(p, Way::ByWeights, cut, stream);
    if (cuts > 0) {
        const i64 blocks = (m * n + 1023) / 1024;
        k_grouped_join<O><<<dim3(static_cast<unsigned>(blocks < 4096 ? blocks : 4096), static_cast<unsigned>(cuts)), 256, 0, stream>>>(
            p.partial, p.plan, p.kinds, p.run, p.m, p.n, p.out, out_stride, out_kind);
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
    const i64 cuts = cuts_of(rows, run_for(rows, outputs, inputs));
    return cuts > 0 ? 4 * 2 * (cuts + 1) * outputs * inputs : 0;
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
