// Products in 8-bit integers with an FP32 scale for each row of both operands (a token of x, a channel of the weights), and the
// kernel that brings rows to that form.
//
//   scale = max(max |x| * c, 2^-126), c = FP32 of 1/127     q = the whole number nearest to x / scale, ties to even
//   out[i][j] = scale_a[i] scale_b[j] sum over k of q_a[i][k] q_b[j][k]
//
// The scale is by definition one product in FP32, not the number nearest to a 127th, from which it is a last place off in one row of
// twenty or so: any scale so near serves as well, but values half a step from a whole number (the largest one's half) go by its
// last place, so a row has one quantisation only where all that bring it to integers form its scale alike.
//
// Sums are of 32-bit integers (v_mfma_i32_16x16x64_i8) and exact up to 2^17 terms (2^17 * 127^2 < 2^31); a product is rounded
// when its sum becomes FP32 and at each scale, by 2^-24 each, and to the output's type.
#include <cmath>

#include "node_tiles.hpp"

namespace smx {
namespace node {
namespace {

constexpr i64 kMostTerms = 1 << 17;

// Quotients are the nearest whole numbers to the exact x / scale: the one from the rounded reciprocal is corrected by the sign
// of what it leaves, r = x - q scale, which is exact in FP32 (a multiple of half the scale's last place, less than the scale).
__device__ __forceinline__ int nearest(float x, float scale, float inverse) {
    float q = rintf(x * inverse);
    const float r = fmaf(-q, scale, x), twice = 2.0f * __builtin_fabsf(r);
    if (twice > scale || (twice == scale && (static_cast<int>(q) & 1))) q += r > 0.0f ? 1.0f : -1.0f;
    return static_cast<int>(q);
}

__device__ __forceinline__ unsigned four(const float* v, float scale, float inverse) {
    unsigned w = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) w |= static_cast<unsigned>(nearest(v[i], scale, inverse) & 0xff) << (8 * i);
    return w;
}

// A row's scale from the largest of its magnitudes' bits (infinities and NaN above all): NaN where the row has one of these.
__device__ __forceinline__ float scale_of_bits(unsigned top) {
    if (top >= 0x7f800000u) return __builtin_nanf("");
    const float scale = __uint_as_float(top) * (1.0f / 127.0f);
    return scale > 0x1p-126f ? scale : 0x1p-126f;
}

// Lanes a row, eight values each at a time; rows of up to 8 LANES PACKS values stay in registers between the largest magnitude and
// the quotients, longer ones (PACKS 0) are read again.  Bytes bound it: 16,384 x 8,192 of bf16 in 85 us, 4.7 TB/s.
template <class T, int LANES, int PACKS>
__global__ void __launch_bounds__(256) k_quantize_integers(const T* __restrict__ x, i64 x_stride, i64 rows, int cols,
                                                           std::int8_t* __restrict__ values, i64 pitch,
                                                           float* __restrict__ scales) {
    __shared__ unsigned room[2][4];
    const int lane = threadIdx.x % LANES;
    int turn = 0;
    for (i64 r = blockIdx.x * (256 / LANES) + threadIdx.x / LANES; r < rows; r += static_cast<i64>(gridDim.x) * (256 / LANES)) {
        const T* const row = x + r * x_stride;
        Eight<T> held[PACKS ? PACKS : 1];
        unsigned top = 0;
        const auto look = [&](const Eight<T>& e) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const unsigned b = __float_as_uint(e[i]) & 0x7fffffffu;
                top = b > top ? b : top;
            }
        };
        if constexpr (PACKS > 0) {
#pragma unroll
            for (int q = 0; q < PACKS; ++q) held[q] = load_pack(row, 8 * (q * LANES + lane), cols);
#pragma unroll
            for (int q = 0; q < PACKS; ++q) {
                settle(held[q], 8 * (q * LANES + lane), cols);
                look(held[q]);
            }
        } else {
            // (columns are counted without a sign: the step past the last one of 2^31 - 513 is past 2^31 too)
            for (unsigned c = 8 * lane; c < static_cast<unsigned>(cols); c += 8 * LANES) {
                Eight<T> e = load_pack(row, static_cast<int>(c), cols);
                settle(e, static_cast<int>(c), cols);
                look(e);
            }
        }
#pragma unroll
        for (int o = 1; o < (LANES < 64 ? LANES : 64); o *= 2) {
            const unsigned other = __shfl_xor(top, o);
            top = other > top ? other : top;
        }
        if constexpr (LANES > 64) {
            // (the two halves of the room in turn: a wave past the barrier may be in its next row while another still reads)
            turn ^= 1;
            if (threadIdx.x % 64 == 0) room[turn][threadIdx.x / 64] = top;
            __syncthreads();
#pragma unroll
            for (int w = 0; w < 4; ++w) top = room[turn][w] > top ? room[turn][w] : top;
        }
        const float scale = scale_of_bits(top);
        if (lane == 0) scales[r] = scale;
        const bool fine = top < 0x7f800000u;
        const float inverse = 1.0f / scale;
        const auto put = [&](const Eight<T>& e, int c) {
            float v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = fine ? e[i] : 0.0f;
            *reinterpret_cast<uint2*>(values + r * pitch + c) =
                fine ? make_uint2(four(v, scale, inverse), four(v + 4, scale, inverse)) : make_uint2(0, 0);
        };
        if constexpr (PACKS > 0) {
#pragma unroll
            for (int q = 0; q < PACKS; ++q) {
                const int c = 8 * (q * LANES + lane);
                if (c < pitch) put(held[q], c);
            }
        } else {
            for (unsigned c = 8 * lane; c < pitch; c += 8 * LANES) {
                Eight<T> e = load_pack(row, static_cast<int>(c), cols);
                settle(e, static_cast<int>(c), cols);
                put(e, static_cast<int>(c));
            }
        }
    }
}

template <class O>
struct Integers {
    const std::int8_t *a, *b;
    const float *as, *bs;
    int m, n, k;
    i64 pitch;
    O* out;
    i64 out_stride;
    int tiles_m, tiles_n;
};

// 2^17 products of -128 by itself, which no row brought to integers here has, are the one sum past 2^31 - 1: as -2^31, which no other
// sum is.
__device__ __forceinline__ float sum_of(int v) { return v == INT32_MIN ? 0x1p31f : static_cast<float>(v); }

// A sum by the row's scale and then by the other.  The scale of a row next to FP32's largest number may take the sum beyond FP32 though
// small weights bring the product back: from 2^96 on it is 2^-32 of itself, and the product 2^32 times what it is then (both exact: the
// sum, a whole number, stays below 2^128, and the product with any second scale above 2^-86).  Few rows are so, and a wave without
// them skips the last step (a choice of the order of the two scales for each value took 8 us of 880 more at 16,384 x 8,192 x 8,192).
template <class O>
__device__ __forceinline__ void store_scaled(const Integers<O>& p, int i, int j, i32x4 v, float a) {
    const bool far = __builtin_fabsf(a) >= 0x1p96f;
    const float by = far ? a * 0x1p-32f : a;
    float o[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) o[q] = sum_of(v[q]) * by * (j + q < p.n ? p.bs[j + q] : 0.0f);
    if (__any(far))
#pragma unroll
        for (int q = 0; q < 4; ++q) o[q] *= far ? 0x1p32f : 1.0f;
    if (i >= p.m) return;
    O* const at = p.out + i * p.out_stride + j;
    if (j + 4 <= p.n) {
        Pack<O, 4> w;
#pragma unroll
        for (int q = 0; q < 4; ++q) w.v[q] = static_cast<O>(o[q]);
        *reinterpret_cast<Pack<O, 4>*>(at) = w;
    } else {
#pragma unroll
        for (int q = 0; q < 4; ++q)
            if (j + q < p.n) at[q] = static_cast<O>(apart(o[q]));
    }
}

template <class O>
__device__ __forceinline__ void store_scaled(const Integers<O>& p, int i, int j, i32x4 v) {
    store_scaled(p, i, j, v, p.as[i < p.m ? i : p.m - 1]);
}

// Tiles as those of 16-bit rows, a step 128 values, both operands by rows.  8192 cubed in 436 us, 2,520 TOP/s (a library's product
// 2,190), the matrix pipe busy 60% of it: a step's fragments and what arrives for the next take LDS about as long as its
// products take the pipe, and a tile's end overlaps with nothing.
template <class O, int BM, int BN, int WM, int WN>
__global__ void __launch_bounds__(64 * WM * WN, BM + BN > 256 ? 1 : 2) k_integer_tiles(Integers<O> p) {
    using T = std::int8_t;
    using A = Step<Lie::Rows, BM, kStepBytes / 2>;
    using B = Step<Lie::Rows, BN, kStepBytes / 2>;
    constexpr int WAVES = WM * WN, NA = A::kPieces / 64 / WAVES, NB = B::kPieces / 64 / WAVES, MF = BM / WM / 16,
                  NF = BN / WN / 16;
    constexpr unsigned kStage = (BM + BN) * kStepBytes;
    __shared__ __attribute__((aligned(1024))) std::uint8_t lds[2 * kStage];
    const unsigned lds0 = static_cast<unsigned>(reinterpret_cast<std::uintptr_t>((__attribute__((address_space(3))) std::uint8_t*)lds));
    const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const int wm = wave / WN * (BM / WM), wn = wave % WN * (BN / WN);
    const int tiles = p.tiles_m * p.tiles_n, steps = static_cast<int>(p.pitch / kStepBytes);
    int i0, j0;
    const T *at_a[NA], *at_b[NB];
    const auto turn_to = [&](int turn) {
        const int id = xcd_remap(turn, tiles);
        const int band = id / (4 * p.tiles_n), in = id % (4 * p.tiles_n);
        const int high = p.tiles_m - 4 * band < 4 ? p.tiles_m - 4 * band : 4;
        i0 = (4 * band + in % high) * BM, j0 = in / high * BN;
#pragma unroll
        for (int q = 0; q < NA; ++q) {
            const int e = (wave + WAVES * q) * 64 + lane, r = i0 + A::row_at(e);
            at_a[q] = p.a + (r < p.m ? r : p.m - 1) * p.pitch + A::piece_at(e) * 16;
        }
#pragma unroll
        for (int q = 0; q < NB; ++q) {
            const int e = (wave + WAVES * q) * 64 + lane, r = j0 + B::row_at(e);
            at_b[q] = p.b + (r < p.n ? r : p.n - 1) * p.pitch + B::piece_at(e) * 16;
        }
    };
    const auto stage = [&](int s, int slot) {
        const unsigned to = __builtin_amdgcn_readfirstlane(lds0 + slot * kStage + wave * 1024);
        each_of<NA>([&](auto q) { fetch<WAVES * q * 1024>(at_a[q] + s * kStepBytes, to); });
        each_of<NB>([&](auto q) { fetch<BM * kStepBytes + WAVES * q * 1024>(at_b[q] + s * kStepBytes, to); });
    };
    int slot = 0;
    turn_to(blockIdx.x);
    stage(0, 0);
    for (int turn = blockIdx.x; turn < tiles; turn += gridDim.x) {
        const int i_now = i0, j_now = j0;
        i32x4 acc[MF][NF];
#pragma unroll
        for (int f = 0; f < MF; ++f)
#pragma unroll
            for (int g = 0; g < NF; ++g) acc[f][g] = i32x4{0, 0, 0, 0};
        for (int s = 0; s < steps; ++s) {
            arrived();
            __syncthreads();
            const std::uint8_t* const tile = lds + slot * kStage;
            slot ^= 1;
            const auto read_a = [&](int f, int q) { return A::read(tile, wm + 16 * f, q, lane); };
            const auto read_b = [&](int g, int q) { return B::read(tile + BM * kStepBytes, wn + 16 * g, q, lane); };
            i32x4 vb[NF], va = read_a(0, 0);
#pragma unroll
            for (int g = 0; g < NF; ++g) vb[g] = read_b(g, 0);
            if (s + 1 < steps) {
                stage(s + 1, slot);
            } else if (turn + static_cast<int>(gridDim.x) < tiles) {
                turn_to(turn + gridDim.x);
                stage(0, slot);
            }
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                // each fragment is read while the one before is multiplied
                i32x4 next_b[NF];
#pragma unroll
                for (int f = 0; f < MF; ++f) {
                    const i32x4 now_a = va;
                    if (f + 1 < MF || q == 0) va = read_a((f + 1) % MF, q + (f + 1) / MF);
                    if (f + 2 == MF && q == 0)
#pragma unroll
                        for (int g = 0; g < NF; ++g) next_b[g] = read_b(g, 1);
#pragma unroll
                    for (int g = 0; g < NF; ++g) acc[f][g] = Multiply<T>::add(vb[g], now_a, acc[f][g]);
                    // (in this order: left to itself the compiler has each read waited for at once)
                    if (f + 1 < MF || q == 0) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
                    if (f + 2 == MF && q == 0) __builtin_amdgcn_sched_group_barrier(0x100, NF, 0);
                    __builtin_amdgcn_sched_group_barrier(0x008, NF, 0);
                }
                if (q == 0)
#pragma unroll
                    for (int g = 0; g < NF; ++g) vb[g] = next_b[g];
            }
        }
        settle_products();
#pragma unroll
        for (int f = 0; f < MF; ++f)
#pragma unroll
            for (int g = 0; g < NF; ++g)
                store_scaled(p, i_now + wm + 16 * f + lane % 16, j_now + wn + 16 * g + 4 * (lane / 16), acc[f][g]);
    }
}

constexpr i64 kFewRows = 16;

// Up to 16 rows: the weights are read once, eight waves share the summed axis, and their sums are added in LDS in order.  The
// weights' bytes bound it: 9 x 4,096 x 8,192 in 8.4 us, 4.0 TB/s.
template <class O>
__global__ void __launch_bounds__(512) k_integer_rows(Integers<O> p) {
    constexpr int NF = 1, KS = 8;
    using T = std::int8_t;
    __shared__ FewRoom<T, NF, KS> room;
    const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), row = lane % 16;
    const int j0 = xcd_remap(blockIdx.x, gridDim.x) * 16 * NF;
    const T* b[NF];
#pragma unroll
    for (int g = 0; g < NF; ++g) {
        const int j = j0 + 16 * g + row;
        b[g] = p.b + (j < p.n ? j : p.n - 1) * p.pitch;
    }
    few_rows<T, true, NF, KS>(p.a + (row < p.m ? row : p.m - 1) * p.pitch, b, static_cast<int>(p.pitch), room);
    for (int g = wave; g < NF; g += KS) store_scaled(p, row, j0 + 16 * g + 4 * (lane / 16), joined(room, g));
}

// Up to kRawRows rows of x as they are given, of up to kRawTerms values: each workgroup brings them to integers itself, in LDS, while its
// first weights are on their way.  One launch in place of two: 1 x 4096 x 8192 in 7.5 us, 10.4 in two.
constexpr int kRawRows = 4, kRawTerms = 8192;

template <class T, class O, int KS>
__global__ void __launch_bounds__(64 * KS) k_integer_raw(Integers<O> p, const T* __restrict__ x, i64 x_stride) {
    constexpr int kAhead = 4, kPacks = kRawTerms / (8 * 64 * KS);
    __shared__ FewRoom<std::int8_t, 1, KS> room;
    __shared__ __attribute__((aligned(16))) std::int8_t brought[kRawRows][kRawTerms];
    __shared__ unsigned tops[kRawRows][KS];
    const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), row = lane % 16;
    const int j0 = xcd_remap(blockIdx.x, gridDim.x) * 16, j = j0 + row < p.n ? j0 + row : p.n - 1;
    const int steps = static_cast<int>(p.pitch / kStepBytes), at = lane / 16 * 16;
    const std::int8_t* const b = p.b + j * p.pitch + at;
    i32x4 wb[kAhead][2];
    const auto load = [&](int s0) {
#pragma unroll
        for (int q = 0; q < kAhead; ++q) {
            const int s = s0 + q * KS < steps ? s0 + q * KS : 0;  // (a step read in vain)
#pragma unroll
            for (int h = 0; h < 2; ++h) wb[q][h] = load_sixteen(b + s * kStepBytes + 64 * h);
        }
    };
    // (x is asked for before the weights: what was asked for first comes first)
    Eight<T> held[kRawRows][kPacks];
#pragma unroll
    for (int r = 0; r < kRawRows; ++r) {
        if (r >= p.m) break;
#pragma unroll
        for (int q = 0; q < kPacks; ++q)
            held[r][q] = load_pack(x + r * x_stride, 8 * (q * 64 * KS + static_cast<int>(threadIdx.x)), p.k);
    }
    __builtin_amdgcn_sched_barrier(0);
    load(wave);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int r = 0; r < kRawRows; ++r) {
        if (r >= p.m) break;
        unsigned top = 0;
#pragma unroll
        for (int q = 0; q < kPacks; ++q) {
            settle(held[r][q], 8 * (q * 64 * KS + static_cast<int>(threadIdx.x)), p.k);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const unsigned bits = __float_as_uint(held[r][q][i]) & 0x7fffffffu;
                top = bits > top ? bits : top;
            }
        }
#pragma unroll
        for (int o = 1; o < 64; o *= 2) {
            const unsigned other = __shfl_xor(top, o);
            top = other > top ? other : top;
        }
        if (lane == 0) tops[r][wave] = top;
    }
    __syncthreads();
    float mine = 0.0f;  // the scale of row lane % 16
#pragma unroll
    for (int r = 0; r < kRawRows; ++r) {
        if (r >= p.m) break;
        unsigned top = 0;
#pragma unroll
        for (int w = 0; w < KS; ++w) top = tops[r][w] > top ? tops[r][w] : top;
        const float scale = scale_of_bits(top), inverse = 1.0f / scale;
        const bool fine = top < 0x7f800000u;
        if (row == r) mine = scale;
#pragma unroll
        for (int q = 0; q < kPacks; ++q) {
            const int c = 8 * (q * 64 * KS + static_cast<int>(threadIdx.x));
            if (c >= p.pitch) break;
            float v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = held[r][q][i];
            *reinterpret_cast<uint2*>(&brought[r][c]) =
                fine ? make_uint2(four(v, scale, inverse), four(v + 4, scale, inverse)) : make_uint2(0, 0);
        }
    }
    __syncthreads();
    i32x4 acc{0, 0, 0, 0};
    for (int s0 = wave; s0 < steps; s0 += KS * kAhead) {
        if (s0 > wave) load(s0);
#pragma unroll
        for (int q = 0; q < kAhead; ++q) {
            if (s0 + q * KS >= steps) break;
#pragma unroll
            for (int h = 0; h < 2; ++h)
                acc = Multiply<std::int8_t>::add(
                    wb[q][h], *reinterpret_cast<const i32x4*>(&brought[row % kRawRows][(s0 + q * KS) * kStepBytes + 64 * h + at]), acc);
            settle_products();  // (the next step is conditional)
        }
    }
    settle_products();
    room.v[wave][0][lane] = acc;
    __syncthreads();
    if (wave > 0) return;
    store_scaled(p, row, j0 + 4 * (lane / 16), joined(room, 0), mine);
}

template <class O>
__global__ void __launch_bounds__(256) k_integer_zero(O* __restrict__ out, i64 out_stride, i64 m, i64 n) {
    for (i64 e = static_cast<i64>(blockIdx.x) * 256 + threadIdx.x; e < m * n; e += static_cast<i64>(gridDim.x) * 256)
        out[e / n * out_stride + e % n] = static_cast<O>(0.0f);
}

void check_sizes(i64 m, i64 n, i64 k) {
    constexpr i64 most = (1LL << 31) - 512;
    require(m >= 0 && m <= most && n >= 0 && n <= most && k >= 0 && k <= most, "sizes must be in [0, 2^31 - 512]");
    if (k > kMostTerms) throw std::domain_error("integer products sum over up to 2^17 values");
}

void check_integers(const void* values, const void* scales, i64 rows, i64 cols, const char* name) {
    if (rows == 0) return;
    if ((cols > 0 && !values) || !scales) throw std::invalid_argument(std::string(name) + " is NULL");
    if (!aligned(values, 16) || !aligned(scales, 4))
        throw std::invalid_argument(std::string(name) + ": integers must be 16-byte aligned, their scales 4-byte");
}

i64 pitch_of(i64 cols) { return (cols + kStepBytes - 1) / kStepBytes * kStepBytes; }

bool raw(i64 m, i64 k) { return m <= kRawRows && k <= kRawTerms; }

template <class T>
void launch_quantize(const T* x, i64 x_stride, i64 rows, i64 cols, std::int8_t* values, float* scales, hipStream_t stream) {
    const i64 pitch = pitch_of(cols);
    const auto go = [&](auto lanes, auto packs) {
        constexpr int L = decltype(lanes)::value, P = decltype(packs)::value;
        const i64 groups = (rows + 256 / L - 1) / (256 / L);
        k_quantize_integers<T, L, P><<<static_cast<unsigned>(groups < 16384 ? groups : 16384), 256, 0, stream>>>(
            x, x_stride, rows, static_cast<int>(cols), values, pitch, scales);
        SMX_LAUNCH_CHECK("k_quantize_integers");
    };
    using std::integral_constant;
    if (pitch <= 128) go(integral_constant<int, 16>{}, integral_constant<int, 1>{});
    else if (pitch <= 512) go(integral_constant<int, 64>{}, integral_constant<int, 1>{});
    else if (pitch <= 1024) go(integral_constant<int, 64>{}, integral_constant<int, 2>{});
    else if (pitch <= 2048) go(integral_constant<int, 256>{}, integral_constant<int, 1>{});
    else if (pitch <= 4096) go(integral_constant<int, 256>{}, integral_constant<int, 2>{});
    else if (pitch <= 8192) go(integral_constant<int, 256>{}, integral_constant<int, 4>{});
    else go(integral_constant<int, 256>{}, integral_constant<int, 0>{});
}

void quantize(const void* x, i64 x_stride, int dtype, i64 rows, i64 cols, std::int8_t* values, float* scales, hipStream_t stream) {
    if (rows == 0) return;
    with_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        launch_quantize(static_cast<const T*>(x), x_stride, rows, cols, values, scales, stream);
    });
}

int tile_for(i64 m, i64 n) {
    const auto rounds = [&](i64 t, i64 held) {
        return ((m + t - 1) / t * ((n + t - 1) / t) + held * kComputeUnits - 1) / (held * kComputeUnits);
    };
    const double t256 = 1.0 * rounds(256, 1), t128 = 1.12 / 2 * rounds(128, 2), t64 = 1.86 / 4 * rounds(64, 4);
    return t256 <= t128 && t256 <= t64 ? 256 : t128 <= t64 ? 128 : 64;
}

template <class O>
Integers<O> integers_of(const std::int8_t* a, const float* as, const std::int8_t* b, const float* bs, i64 m, i64 n, i64 k, O* out,
                        i64 out_stride) {
    Integers<O> p{};
    p.a = a, p.as = as, p.b = b, p.bs = bs;
    p.m = static_cast<int>(m), p.n = static_cast<int>(n), p.k = static_cast<int>(k);
    p.pitch = pitch_of(k);
    p.out = out, p.out_stride = out_stride;
    return p;
}

// f(q) for columns of p that one launch of few rows takes: it has 512 threads for each 16, and a launch fewer than 2^32.
constexpr i64 kColumnsOnce = 1 << 26;

template <class O, class F>
void each_slice(const Integers<O>& p, F&& f) {
    for (i64 j = 0; j < p.n; j += kColumnsOnce) {
        Integers<O> q = p;
        q.b += j * p.pitch, q.bs += j, q.out += j;
        q.n = static_cast<int>(p.n - j < kColumnsOnce ? p.n - j : kColumnsOnce);
        f(q);
    }
}

template <class O>
void launch_product(const std::int8_t* a, const float* as, const std::int8_t* b, const float* bs, i64 m, i64 n, i64 k, O* out,
                    i64 out_stride, hipStream_t stream) {
    if (k == 0) {
        k_integer_zero<O><<<static_cast<unsigned>(m * n < 256 * 4096 ? (m * n + 255) / 256 : 4096), 256, 0, stream>>>(
            out, out_stride, m, n);
        SMX_LAUNCH_CHECK("k_integer_zero");
        return;
    }
    Integers<O> p = integers_of(a, as, b, bs, m, n, k, out, out_stride);
    if (m <= kFewRows) {
        each_slice(p, [&](const Integers<O>& q) {
            k_integer_rows<O><<<blocks_for(q.n, 16), 512, 0, stream>>>(q);
            SMX_LAUNCH_CHECK("k_integer_rows");
        });
        return;
    }
    const i64 t = tile_for(m, n), tiles_m = (m + t - 1) / t, tiles_n = (n + t - 1) / t;
    require(tiles_m * tiles_n < (1LL << 31) && 8 * tiles_n < (1LL << 31), "the product has too many tiles");
    p.tiles_m = static_cast<int>(tiles_m), p.tiles_n = static_cast<int>(tiles_n);
    const auto grid = [&](i64 held) {
        const i64 most = held * kComputeUnits;
        return static_cast<unsigned>(tiles_m * tiles_n < most ? tiles_m * tiles_n : most);
    };
    switch (t) {
        case 256: k_integer_tiles<O, 256, 256, 2, 4><<<grid(1), 512, 0, stream>>>(p); break;
        case 128: k_integer_tiles<O, 128, 128, 2, 2><<<grid(2), 256, 0, stream>>>(p); break;
        default: k_integer_tiles<O, 64, 64, 2, 2><<<grid(4), 256, 0, stream>>>(p);
    }
    SMX_LAUNCH_CHECK("k_integer_tiles");
}

}  // namespace
}  // namespace node
}  // namespace smx

using namespace smx;
using namespace smx::node;

extern "C" {

int64_t smx_integer_stride(int64_t cols) { return cols > 0 ? pitch_of(cols) : 0; }

int32_t smx_integer_quantize(const void* x, int64_t x_stride, int32_t dtype, int64_t rows, int64_t cols, int8_t* values,
                             float* scales, void* stream) {
    return guarded([&] {
        check_sizes(rows, 0, 0);
        require(cols >= 0 && cols < (1LL << 31) - 512, "sizes must be in [0, 2^31 - 512)");
        require(dtype >= SMX_DTYPE_F32 && dtype <= SMX_DTYPE_F16, "unknown dtype code");
        check_rows(x, x_stride, rows, cols, dtype, "x");
        check_integers(values, scales, rows, cols, "values");
        quantize(x, x_stride, dtype, rows, cols, values, scales, static_cast<hipStream_t>(stream));
    });
}

int32_t smx_integer_product(const int8_t* a_values, const float* a_scales, const int8_t* b_values, const float* b_scales, int64_t m,
                            int64_t n, int64_t k, int32_t dtype, void* out, int64_t out_stride, void* stream) {
    return guarded([&] {
        check_sizes(m, n, k);
        require(dtype >= SMX_DTYPE_F32 && dtype <= SMX_DTYPE_F16, "unknown dtype code");
        check_integers(a_values, a_scales, m, k, "a");
        check_integers(b_values, b_scales, n, k, "b");
        check_rows(out, out_stride, m, n, dtype, "out");
        if (m == 0 || n == 0) return;
        with_dtype(dtype, [&](auto o) {
            using O = decltype(o);
            launch_product<O>(a_values, a_scales, b_values, b_scales, m, n, k, static_cast<O*>(out), out_stride,
                              static_cast<hipStream_t>(stream));
        });
    });
}

int64_t smx_integer_linear_workspace(int64_t m, int64_t n, int64_t k) {
    return m > 0 && n > 0 && k > 0 && !raw(m, k) ? m * pitch_of(k) + 4 * m : 0;
}

int32_t smx_integer_linear(const void* x, int64_t x_stride, int32_t dtype, const int8_t* w_values, const float* w_scales, int64_t m,
                           int64_t n, int64_t k, int32_t out_dtype, void* out, int64_t out_stride, void* workspace,
                           int64_t workspace_bytes, void* stream) {
    return guarded([&] {
        check_sizes(m, n, k);
        require(dtype >= SMX_DTYPE_F32 && dtype <= SMX_DTYPE_F16, "unknown dtype code");
        require(out_dtype >= SMX_DTYPE_F32 && out_dtype <= SMX_DTYPE_F16, "unknown dtype code");
        check_rows(x, x_stride, m, k, dtype, "x");
        check_integers(w_values, w_scales, n, k, "w");
        check_rows(out, out_stride, m, n, out_dtype, "out");
        check_workspace(workspace, workspace_bytes, smx_integer_linear_workspace(m, n, k));
        if (m == 0 || n == 0) return;
        if (k > 0 && raw(m, k)) {
            with_dtype(dtype, [&](auto t) {
                with_dtype(out_dtype, [&](auto o) {
                    using T = decltype(t);
                    using O = decltype(o);
                    const auto p = integers_of<O>(nullptr, nullptr, w_values, w_scales, m, n, k, static_cast<O*>(out), out_stride);
                    each_slice(p, [&](const Integers<O>& q) {
                        k_integer_raw<T, O, 8><<<blocks_for(q.n, 16), 512, 0, static_cast<hipStream_t>(stream)>>>(
                            q, static_cast<const T*>(x), x_stride);
                        SMX_LAUNCH_CHECK("k_integer_raw");
                    });
                });
            });
            return;
        }
        auto* const values = static_cast<std::int8_t*>(workspace);
        auto* const scales = k > 0 ? reinterpret_cast<float*>(values + m * pitch_of(k)) : nullptr;
        if (k > 0) quantize(x, x_stride, dtype, m, k, values, scales, static_cast<hipStream_t>(stream));
        with_dtype(out_dtype, [&](auto o) {
            using O = decltype(o);
            launch_product<O>(values, scales, w_values, w_scales, m, n, k, static_cast<O*>(out), out_stride,
                              static_cast<hipStream_t>(stream));
        });
    });
}

}  // extern "C"
