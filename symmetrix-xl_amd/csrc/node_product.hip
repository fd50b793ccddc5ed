// Matrix products of E4M3 values with an E8M0 scale for each block of 128 values
// along the summed axis, and the kernels that bring matrices to that form.
//
// Two forms of the product, both with FP32 accumulators:
//   - 8-bit: v_mfma_scale_f32_16x16x128_f8f6f4 sums one block of 128 and applies both operands'
//     scales, powers of two, by itself.  Its adder aligns eight products to the largest of them
//     and drops what lies below 2^-13 of that one (measured: 2^16 + 127 products of 2^2 comes out
//     28 short, those of 2^4 exact): 2^-16 of an output's norm in rows of normal values, however long, and at most
//     7 x 2^-13 of the largest of each eight.
//   - bf16: an E4M3 value times its scale is a bf16 value exactly (v_cvt_scalef32_pk_bf16_fp8), and
//     v_mfma_f32_16x16x32_bf16 sums as FP32 does, 2^-24 to 2^-27 of the norm there, at half the rate.  (Values below
//     2^-126 are bf16's subnormal numbers, multiples of 2^-133; the instructions keep these.)
// FP32 outputs take the bf16 form, so that their sums are FP32 sums.  16-bit outputs, which are rounded
// to 2^-9 or 2^-12 anyway, take the 8-bit form, but for short sums (up to 256), where what the adder drops is as much as FP32
// sums may be off, (k + 8) 2^-23 of the terms' magnitudes, or more (1.3 times that at 128 terms, 0.36 at 256): 20000 x 1024 x
// 256 16.4 us in the bf16 form, 13.3 in the 8-bit one; x 512 25.0 and 18.3.
#include "node_ops.hpp"

namespace smx {
namespace node {
namespace {

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

constexpr i64 kShortSum = 256;

// Blocks along the rows: 16 lanes a block, eight values each, so a row's loads
// and stores are whole lines.  One read of x and one write of a byte a value, at 5.1 TB/s (16384 x 8192 bf16, 79 us).
template <class T>
__global__ void __launch_bounds__(256) k_quantize_rows(const T* __restrict__ x, i64 x_stride, i64 rows, i64 cols,
                                                       std::uint8_t* __restrict__ values,
                                                       std::uint8_t* __restrict__ scales, i64 pitch, i64 scale_pitch) {
    const int sub = threadIdx.x % 16;
    const unsigned blocks = static_cast<unsigned>(pitch / kBlock);
    for (i64 g = static_cast<i64>(blockIdx.x) * 16 + threadIdx.x / 16; g < rows * blocks;
         g += static_cast<i64>(gridDim.x) * 16) {
        const i64 r = g < (1LL << 32) ? static_cast<unsigned>(g) / blocks : g / blocks;
        const int k = static_cast<int>(g - r * blocks);
        const int c = k * kBlock + 8 * sub;
        float v[8];
        load_eight(x + r * x_stride, c, static_cast<int>(cols), v);
        const int byte = block_scale_byte(row_max(top_of(v)));
        *reinterpret_cast<uint2*>(values + r * pitch + c) = e4m3_eight(v, block_inverse_scale(byte));
        std::uint8_t* const sc = scales + r * scale_pitch + k;
        if (sub == 0) *sc = static_cast<std::uint8_t>(byte);
        if (k + 1 == static_cast<int>(blocks) && sub > 0 && k + sub < scale_pitch) sc[sub] = 0;
    }
}

// One tile of 128 x 128 a workgroup: blocks along its columns, stored as rows of
// the transpose, and along its rows too (ROWS) in the same reading.  A thread
// holds 8 x 8 values; the transposed bytes cross LDS in pieces of eight, each column's
// pieces permuted by the column so that the 16 lanes that write at once meet 16 places.  16384 x 8192 bf16 to both: 129 us,
// 4.2 TB/s, against 79 us and another reading for each alone.
template <class T, bool ROWS>
__global__ void __launch_bounds__(256) k_quantize_tile(const T* __restrict__ x, i64 x_stride, i64 rows, i64 cols,
                                                       std::uint8_t* __restrict__ values,
                                                       std::uint8_t* __restrict__ scales, i64 pitch, i64 scale_pitch,
                                                       std::uint8_t* __restrict__ values_t,
                                                       std::uint8_t* __restrict__ scales_t, i64 pitch_t,
                                                       i64 scale_pitch_t) {
    __shared__ float tops[16][kBlock + 4];
    __shared__ int bytes[kBlock];
    __shared__ uint2 turned[kBlock][16];
    const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
    const i64 blocks_c = (cols + kBlock - 1) / kBlock;
    const i64 tr = blockIdx.x / blocks_c, tc = blockIdx.x % blocks_c;
    const i64 r0 = tr * kBlock + 8 * ty, c0 = tc * kBlock + 8 * tx;
    Eight<T> in[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        if (r0 + i < rows) {
            in[i] = load_pack(x + (r0 + i) * x_stride, static_cast<int>(c0), static_cast<int>(cols));
        } else {
#pragma unroll
            for (int j = 0; j < Eight<T>::kWords; ++j) in[i].w[j] = 0;
        }
    }
    float v[8][8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        settle(in[i], static_cast<int>(c0), static_cast<int>(cols));
#pragma unroll
        for (int j = 0; j < 8; ++j) v[i][j] = in[i][j];
    }
    if constexpr (ROWS) {
        const int k = static_cast<int>(tc);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int byte = block_scale_byte(row_max(top_of(v[i])));
            if (r0 + i >= rows) continue;
            *reinterpret_cast<uint2*>(values + (r0 + i) * pitch + c0) = e4m3_eight(v[i], block_inverse_scale(byte));
            std::uint8_t* const sc = scales + (r0 + i) * scale_pitch + k;
            if (tx == 0) *sc = static_cast<std::uint8_t>(byte);
            if (tc + 1 == blocks_c && tx > 0 && k + tx < scale_pitch) sc[tx] = 0;
        }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        float top = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) top = fmaxf(top, finite_magnitude(v[i][j]));
        tops[ty][8 * tx + j] = top;
    }
    __syncthreads();
    if (threadIdx.x < kBlock) {
        float top = 0.0f;
#pragma unroll
        for (int i = 0; i < 16; ++i) top = fmaxf(top, tops[i][threadIdx.x]);
        const int byte = block_scale_byte(top);
        bytes[threadIdx.x] = byte;
        const i64 c = tc * kBlock + threadIdx.x;
        if (c < cols) {
            std::uint8_t* const sc = scales_t + c * scale_pitch_t + tr;
            *sc = static_cast<std::uint8_t>(byte);
            if ((tr + 1) * kBlock >= rows)
                for (i64 z = tr + 1; z < scale_pitch_t; ++z) sc[z - tr] = 0;
        }
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        float w[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = v[i][j];
        turned[8 * tx + j][ty ^ tx] = e4m3_eight(w, block_inverse_scale(bytes[8 * tx + j]));
    }
    __syncthreads();
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const int p = q * 256 + threadIdx.x, c = p / 8, piece = p % 8 * 2;
        const uint2 lo = turned[c][piece ^ (c / 8)], hi = turned[c][(piece + 1) ^ (c / 8)];
        if (tc * kBlock + c < cols)
            *reinterpret_cast<uint4*>(values_t + (tc * kBlock + c) * pitch_t + tr * kBlock + 8 * piece) =
                make_uint4(lo.x, lo.y, hi.x, hi.y);
    }
}

// The accumulators of a chain of MFMAs are read by other instructions right after it;
// eighteen wait states on every path into what follows (the 16x16x128 form takes
// eight passes), with the scheduler fenced on both sides.
__device__ __forceinline__ void mfma_settle() {
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_nop 8\n\ts_nop 8");
    __builtin_amdgcn_sched_barrier(0);
}

// Eight E4M3 values (two dwords) times a scale, as bf16.
__device__ __forceinline__ bf16x8 to_bf16(int lo, int hi, float scale) {
    const bf16x2 p[4] = {__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, false),
                         __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, true),
                         __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, false),
                         __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, true)};
    return __builtin_shufflevector(__builtin_shufflevector(p[0], p[1], 0, 1, 2, 3),
                                   __builtin_shufflevector(p[2], p[3], 0, 1, 2, 3), 0, 1, 2, 3, 4, 5, 6, 7);
}

// 2^(byte - 127) as a float
__device__ __forceinline__ float scale_of(int byte) {
    return byte ? __uint_as_float(static_cast<unsigned>(byte) << 23) : 0x1p-127f;
}

// Operands and output of one product, the rows of both operands in 8-bit blocks.
template <class O>
struct Product {
    const std::uint8_t *a, *as, *b, *bs;
    int m, n;
    int blocks;  // of 128 along the summed axis
    i64 pitch, scale_pitch;
    O* out;
    i64 out_stride;
    float* partial;  // [splits][m][n] when the sum is split, else NULL
    int split_blocks;
    int tiles_m, tiles_n;
};

// A lane's four neighbouring outputs of row i from column j on.
template <class O>
__device__ __forceinline__ void store_four(const Product<O>& p, int i, int j, acc4 v, int split) {
    if (i >= p.m) return;
    if (p.partial) {
        float* const at = p.partial + (static_cast<i64>(split) * p.m + i) * p.n + j;
        if (p.n % 4 == 0 && j + 4 <= p.n) {
            *reinterpret_cast<acc4*>(at) = v;
        } else {
#pragma unroll
            for (int q = 0; q < 4; ++q)
                if (j + q < p.n) at[q] = apart(v[q]);
        }
        return;
    }
    O* const at = p.out + i * p.out_stride + j;
    if (j + 4 <= p.n) {
        Pack<O, 4> o;
#pragma unroll
        for (int q = 0; q < 4; ++q) o.v[q] = static_cast<O>(v[q]);
        *reinterpret_cast<Pack<O, 4>*>(at) = o;
    } else {
#pragma unroll
        for (int q = 0; q < 4; ++q)
            if (j + q < p.n) at[q] = static_cast<O>(apart(v[q]));
    }
}

// Sixteen bytes of neighbouring outputs of row i from column j on.
template <class O>
__device__ __forceinline__ void store_sixteen(const Product<O>& p, int i, int j, i32x4 v) {
    constexpr int kValues = 16 / sizeof(O);
    struct __attribute__((packed, aligned(sizeof(O)))) Words {
        i32x4 w;
    };
    if (i >= p.m) return;
    O* const at = p.out + i * p.out_stride + j;
    if (j + kValues <= p.n) {
        reinterpret_cast<Words*>(at)->w = v;
        return;
    }
    union {
        i32x4 w;
        O o[kValues];
    } parts;
    asm volatile("" : "+v"(v));  // (apart from the whole store)
    parts.w = v;
#pragma unroll
    for (int q = 0; q < kValues; ++q)
        if (j + q < p.n) at[q] = parts.o[q];
}

// 1 KB of LDS at byte `lds` (the wave's own, uniform) from 64 lanes' 16 bytes at their offsets `at`
// into the buffer: memory to LDS without registers.  The compiler does not count it: dma_wait.
__device__ __forceinline__ void dma(__amdgpu_buffer_rsrc_t from, unsigned lds, int at, int also) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds"
                 :
                 : "s"(lds), "v"(at), "s"(from), "s"(also)
                 : "memory");
}
// 256 bytes, four a lane, as above.
__device__ __forceinline__ void dma_words(__amdgpu_buffer_rsrc_t from, unsigned lds, int at, int also) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dword %1, %2, %3 offen lds"
                 :
                 : "s"(lds), "v"(at), "s"(from), "s"(also)
                 : "memory");
}
__device__ __forceinline__ void dma_wait() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

// BM x BN outputs a workgroup of WM x WN x KG waves.  Both operands' blocks of 128
// go to LDS by dma, KG blocks at a time: while some are multiplied, the next ones
// arrive.  A row's eight 16-byte pieces are permuted by half the row's number (in the global
// addresses, within one line), so that the 16 rows that a fragment read meets at once lie in
// 16 different places of the 64 banks.  Lane l holds row l % 16 of a fragment and pieces l / 16 and
// l / 16 + 4 of the block: the order of k inside a block is the operands' own affair, as one
// scale covers it.  The accumulator's lane l holds column l % 16 of rows 4 (l / 16) on; with b as the first operand its
// four values lie side by side in a row of the output.  With KG == 1 a workgroup goes through every gridDim.x-th
// tile, and the next one's first blocks arrive while this one's last are multiplied and stored.  With KG > 1, for
// few tiles, KG groups of waves take every KG-th block each, so that their waits overlap, and their sums are joined in LDS.
// Large products: 16384 x 8192 x 8192 in 855 us, 2,570 TFLOP/s (a library's product of 8-bit values with one scale
// reached 2,880): the matrix pipes are busy 57% of the cycles at the 1.8 GHz that the clock falls to, LDS instructions 23%,
// without bank conflicts (counted).  Neither is full; what is left, by exclusion, are the waits at each step's barrier, which
// one workgroup a unit has no other work to cover with.
// To FP32 8192 cubed takes 767 us, 1,433 TFLOP/s (a library's bf16 product 1,406).
template <class O, bool WIDE, int BM, int BN, int WM, int WN, int KG>
__global__ void __launch_bounds__(64 * WM * WN * KG, (BM + BN) * kBlock * KG * 2 > 81920 ? 1 : 2)
k_product_tile(Product<O> p) {
    constexpr int WAVES = WM * WN * KG, MF = BM / WM / 16, NF = BN / WN / 16, LA = BM / 8 * KG / WAVES,
                  LB = BN / 8 * KG / WAVES, LS = ((BM + BN) / 64 + WAVES - 1) / WAVES;
    constexpr unsigned kOne = (BM + BN) * kBlock, kStage = kOne * KG, kScales = 2 * kStage;
    static_assert(BM * KG % (8 * WAVES) == 0 && BN * KG % (8 * WAVES) == 0 && BM % 64 == 0 && BN % 64 == 0 && 4 % KG == 0);
    static_assert(KG == 1 || 2 * kStage >= WAVES * MF * NF * 1024);
    __shared__ __attribute__((aligned(1024))) std::uint8_t lds[2 * kStage + 8 * (BM + BN)];
    const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const int kg = wave / (WM * WN), in_group = wave % (WM * WN);
    const int wm = in_group / WN * (BM / WM), wn = in_group % WN * (BN / WN);
    const int tiles = p.tiles_m * p.tiles_n;
    const int first = blockIdx.y * p.split_blocks;
    const int last = first + p.split_blocks < p.blocks ? first + p.split_blocks : p.blocks;
    const int pitch = static_cast<int>(p.pitch), scale_pitch = static_cast<int>(p.scale_pitch);
    const unsigned lds0 = static_cast<unsigned>(reinterpret_cast<std::uintptr_t>(
        (__attribute__((address_space(3))) std::uint8_t*)lds));

    // The tile whose blocks are being read.  Bands of four tile rows, each band column by column: the
    // tiles that one XCD works on share their rows of both operands in its L2.  (What a group reads past the
    // last block, within the buffers' ranges, is not used.)
    __amdgpu_buffer_rsrc_t ra, rb, rs[LS];
    int i0, j0, at_a[LA], at_b[LB], at_s[LS];
    const auto turn_to = [&](int turn) {
        const int id = xcd_remap(turn, tiles);
        const int band = id / (4 * p.tiles_n), in_band = id % (4 * p.tiles_n);
        const int high = p.tiles_m - 4 * band < 4 ? p.tiles_m - 4 * band : 4;
        i0 = (4 * band + in_band % high) * BM, j0 = in_band / high * BN;
        const int rows_a = p.m - i0 < BM ? p.m - i0 : BM, rows_b = p.n - j0 < BN ? p.n - j0 : BN;
        ra = __builtin_amdgcn_make_buffer_rsrc(const_cast<std::uint8_t*>(p.a + i0 * p.pitch), 0, rows_a * pitch, 0x00020000);
        rb = __builtin_amdgcn_make_buffer_rsrc(const_cast<std::uint8_t*>(p.b + j0 * p.pitch), 0, rows_b * pitch, 0x00020000);
#pragma unroll
        for (int q = 0; q < LA; ++q) {
            const int w = wave + WAVES * q, r = 8 * (w % (BM / 8)) + lane / 8;
            at_a[q] = (r < rows_a ? r : rows_a - 1) * pitch + ((lane % 8) ^ (r / 2 % 8)) * 16 + w / (BM / 8) * kBlock;
        }
#pragma unroll
        for (int q = 0; q < LB; ++q) {
            const int w = wave + WAVES * q, r = 8 * (w % (BN / 8)) + lane / 8;
            at_b[q] = (r < rows_b ? r : rows_b - 1) * pitch + ((lane % 8) ^ (r / 2 % 8)) * 16 + w / (BN / 8) * kBlock;
        }
        // The scales of four blocks are one dword a row, which goes to LDS the same way, 64 rows an
        // instruction, while the four blocks before are worked on.
#pragma unroll
        for (int q = 0; q < LS; ++q) {
            const int w = wave + WAVES * q, rows = w < BM / 64 ? rows_a : rows_b;
            rs[q] = __builtin_amdgcn_make_buffer_rsrc(
                const_cast<std::uint8_t*>(w < BM / 64 ? p.as + i0 * p.scale_pitch : p.bs + j0 * p.scale_pitch), 0,
                rows * scale_pitch, 0x00020000);
            const int r = 64 * (w < BM / 64 ? w : w - BM / 64) + lane;
            at_s[q] = (r < rows ? r : rows - 1) * scale_pitch;
        }
    };
    const auto stage = [&](int kb, int slot) {
        const unsigned to = __builtin_amdgcn_readfirstlane(lds0 + slot * kStage);
#pragma unroll
        for (int q = 0; q < LA; ++q) {
            const int w = wave + WAVES * q;
            dma(ra, to + w / (BM / 8) * kOne + w % (BM / 8) * 1024, at_a[q], kb * kBlock);
        }
#pragma unroll
        for (int q = 0; q < LB; ++q) {
            const int w = wave + WAVES * q;
            dma(rb, to + w / (BN / 8) * kOne + BM * kBlock + w % (BN / 8) * 1024, at_b[q], kb * kBlock);
        }
    };
    const auto stage_scales = [&](int group, int slot) {
        const unsigned to = __builtin_amdgcn_readfirstlane(lds0 + kScales + slot * (BM + BN) * 4);
#pragma unroll
        for (int q = 0; q < LS; ++q)
            if (wave + WAVES * q < (BM + BN) / 64) dma_words(rs[q], to + 256 * (wave + WAVES * q), at_s[q], 4 * group);
    };

    const int piece = (lane % 16) * kBlock + ((lane / 16) ^ (lane % 16 / 2)) * 16;
    int slot = 0, scale_slot = 0;
    turn_to(blockIdx.x);
    stage_scales(first / 4, 0);
    stage(first, 0);
    for (int turn = blockIdx.x; turn < tiles; turn += gridDim.x) {
        const int i_now = i0, j_now = j0;
        acc4 acc[MF][NF];
#pragma unroll
        for (int f = 0; f < MF; ++f)
#pragma unroll
            for (int g = 0; g < NF; ++g) acc[f][g] = acc4{0.0f, 0.0f, 0.0f, 0.0f};
        unsigned sa[MF], sb[NF];
        for (int kb = first; kb < last; kb += KG) {
            dma_wait();
            __syncthreads();  // the blocks are there, and all have read the ones before
            if (kb % 4 == 0) {
                const unsigned* const now = reinterpret_cast<const unsigned*>(lds + kScales) + scale_slot * (BM + BN) + lane % 16;
#pragma unroll
                for (int f = 0; f < MF; ++f) sa[f] = now[wm + 16 * f] >> (8 * kg);
#pragma unroll
                for (int g = 0; g < NF; ++g) sb[g] = now[BM + wn + 16 * g] >> (8 * kg);
                scale_slot ^= 1;
                if (kb + 4 < last) stage_scales(kb / 4 + 1, scale_slot);
            }
            const std::uint8_t* const tile = lds + slot * kStage + kg * kOne;
            slot ^= 1;
            if (KG == 1 || kb + kg < last) {
                const auto fragment = [&](int row) {
                    const i32x4 x = *reinterpret_cast<const i32x4*>(tile + row * kBlock + piece);
                    const i32x4 y = *reinterpret_cast<const i32x4*>(tile + row * kBlock + (piece ^ 64));
                    return __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7);
                };
                i32x8 vb[NF];
#pragma unroll
                for (int g = 0; g < NF; ++g) vb[g] = fragment(BM + wn + 16 * g);
                if (kb + KG < last) {
                    stage(kb + KG, slot);
                } else if (KG == 1 && turn + static_cast<int>(gridDim.x) < tiles) {
                    turn_to(turn + gridDim.x);
                    stage_scales(first / 4, scale_slot);
                    stage(first, slot);
                }
                if constexpr (!WIDE) {
#pragma unroll
                    for (int f = 0; f < MF; ++f) {
                        const i32x8 va = fragment(wm + 16 * f);
#pragma unroll
                        for (int g = 0; g < NF; ++g)
                            acc[f][g] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(vb[g], va, acc[f][g], 0, 0, 0,
                                                                                        sb[g], 0, sa[f]);
                    }
                } else {
                    i32x8 va[MF];
#pragma unroll
                    for (int f = 0; f < MF; ++f) va[f] = fragment(wm + 16 * f);
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        bf16x8 wb[NF];
#pragma unroll
                        for (int g = 0; g < NF; ++g)
                            wb[g] = to_bf16(vb[g][2 * q], vb[g][2 * q + 1], scale_of(sb[g] & 0xff));
#pragma unroll
                        for (int f = 0; f < MF; ++f) {
                            const bf16x8 wa = to_bf16(va[f][2 * q], va[f][2 * q + 1], scale_of(sa[f] & 0xff));
#pragma unroll
                            for (int g = 0; g < NF; ++g)
                                acc[f][g] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wb[g], wa, acc[f][g], 0, 0, 0);
                        }
                    }
                }
                if constexpr (KG > 1) mfma_settle();  // (the block is conditional)
            }
#pragma unroll
            for (int f = 0; f < MF; ++f) sa[f] = KG < 4 ? sa[f] >> (8 * KG) : 0;
#pragma unroll
            for (int g = 0; g < NF; ++g) sb[g] = KG < 4 ? sb[g] >> (8 * KG) : 0;
        }
        mfma_settle();
        const auto put = [&](int f, int g, acc4 v) {
            store_four(p, i_now + wm + 16 * f + lane % 16, j_now + wn + 16 * g + 4 * (lane / 16), v, blockIdx.y);
        };
        if constexpr (KG == 1) {
            if (sizeof(O) == 4 || p.partial) {
#pragma unroll
                for (int f = 0; f < MF; ++f)
#pragma unroll
                    for (int g = 0; g < NF; ++g) put(f, g, acc[f][g]);
                continue;
            }
            // Values of two bytes go through LDS (the last blocks' place, once all have read them), 16 rows at a time,
            // so that a store is of sixteen bytes a lane and whole lines: 20000 x 1024 x 512 in 17.9 us, 20.9 without.
            constexpr int kRow = 16 * NF * sizeof(O) + 16, kLanes = NF * sizeof(O);
            static_assert(sizeof(O) == 4 || WAVES * 16 * kRow <= kStage);
            std::uint8_t* const room = lds + (slot ^ 1) * kStage + wave * 16 * kRow;
            __syncthreads();
#pragma unroll
            for (int f = 0; f < MF; ++f) {
#pragma unroll
                for (int g = 0; g < NF; ++g) {
                    Pack<O, 4> o;
#pragma unroll
                    for (int q = 0; q < 4; ++q) o.v[q] = static_cast<O>(acc[f][g][q]);
                    __builtin_memcpy(__builtin_assume_aligned(
                                         room + lane % 16 * kRow + (16 * g + 4 * (lane / 16)) * sizeof(O), 4 * sizeof(O)),
                                     &o, sizeof(o));
                }
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
                for (int q = 0; q < kLanes / 4; ++q) {
                    const int r = lane / kLanes + 64 / kLanes * q, c = lane % kLanes;
                    store_sixteen(p, i_now + wm + 16 * f + r, j_now + wn + c * static_cast<int>(16 / sizeof(O)),
                                  *reinterpret_cast<const i32x4*>(room + r * kRow + 16 * c));
                }
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            }
        } else {
            // fragment q of every group is added up, in the groups' order, by group q % KG
            acc4* const room = reinterpret_cast<acc4*>(lds);
            const auto at = [&](int group, int q) {
                return room + ((group * WM * WN + in_group) * MF * NF + q) * 64 + lane;
            };
            __syncthreads();
#pragma unroll
            for (int q = 0; q < MF * NF; ++q) *at(kg, q) = acc[q / NF][q % NF];
            __syncthreads();
#pragma unroll
            for (int q = 0; q < MF * NF; ++q) {
                if (q % KG != kg) continue;
                acc4 sum = *at(0, q);
#pragma unroll
                for (int h = 1; h < KG; ++h) sum += *at(h, q);
                put(q / NF, q % NF, sum);
            }
        }
    }
}

// Rows that k_product_rows takes, and those up to which its waves bring x to 8 bits themselves: that
// work is done again for every 16 or 32 columns.
constexpr i64 kFewRows = 16;
constexpr int kRawRows = 4;

// Up to 16 rows of a: 16 NF columns a workgroup, its KS waves every KS-th block each, joined in LDS.  The
// weights' bytes are all of it, so they go straight to registers, kAhead blocks of them under way at once; a
// wave brings its blocks of x to 8 bits itself (RAW: up to kRawRows rows of x as they are given), eight values a lane, which
// cross LDS to the lanes of the fragment.  Fragment rows past the last row hold some row again and are not stored.
template <class T, class O, bool RAW, bool WIDE, int NF, int KS>
__global__ void __launch_bounds__(64 * KS) k_product_rows(Product<O> p, const T* __restrict__ x, i64 x_stride, int k) {
    constexpr int kAhead = 4;
    __shared__ acc4 room[KS][NF][64];
    __shared__ __attribute__((aligned(16))) std::uint8_t brought[RAW ? KS : 1][RAW ? kAhead : 1][kRawRows * kBlock];
    __shared__ int brought_scale[RAW ? KS : 1][RAW ? kAhead : 1][kRawRows];
    // (a wave's branches have to be the whole wave's to the compiler too: matrix instructions run for all lanes)
    const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const int row = lane % 16, at = lane / 16 * 16;
    const int j0 = xcd_remap(blockIdx.x, gridDim.x) * 16 * NF;
    const std::uint8_t *b[NF], *bs[NF];
#pragma unroll
    for (int g = 0; g < NF; ++g) {
        const int j = j0 + 16 * g + row < p.n ? j0 + 16 * g + row : p.n - 1;
        b[g] = p.b + j * p.pitch + at;
        bs[g] = p.bs + j * p.scale_pitch;
    }
    const int ia = row < p.m ? row : p.m - 1;
    const int from = lane / 16 < p.m ? lane / 16 : p.m - 1;  // RAW: the row and values that this lane brings
    const T* const xr = RAW ? x + from * x_stride : nullptr;
    const std::uint8_t* const ar = RAW ? nullptr : p.a + ia * p.pitch + at;
    acc4 acc[NF];
#pragma unroll
    for (int g = 0; g < NF; ++g) acc[g] = acc4{0.0f, 0.0f, 0.0f, 0.0f};
    for (int kb0 = wave; kb0 < p.blocks; kb0 += KS * kAhead) {
        i32x4 wb[kAhead][NF][2], wa[kAhead][2];
        int sb[kAhead][NF], sa[kAhead];
        Eight<T> v[kAhead];
#pragma unroll
        for (int q = 0; q < kAhead; ++q) {
            const int kb = kb0 + q * KS < p.blocks ? kb0 + q * KS : kb0;  // (a block read twice is used once)
#pragma unroll
            for (int g = 0; g < NF; ++g) {
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    wb[q][g][h] = *reinterpret_cast<const i32x4*>(b[g] + static_cast<i64>(kb) * kBlock + 64 * h);
                sb[q][g] = bs[g][kb];
            }
            if constexpr (RAW) {
                v[q] = load_pack(xr, kb * kBlock + 8 * row, k);
            } else {
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    wa[q][h] = *reinterpret_cast<const i32x4*>(ar + static_cast<i64>(kb) * kBlock + 64 * h);
                sa[q] = p.as[ia * p.scale_pitch + kb];
            }
        }
#pragma unroll
        for (int q = 0; q < kAhead; ++q) {
            if constexpr (RAW) {
                const int kb = kb0 + q * KS < p.blocks ? kb0 + q * KS : kb0;
                settle(v[q], kb * kBlock + 8 * row, k);
                float f[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) f[i] = v[q][i];
                const int byte = block_scale_byte(row_max(top_of(f)));
                *reinterpret_cast<uint2*>(&brought[wave][q][8 * lane]) = e4m3_eight(f, block_inverse_scale(byte));
                if (row == 0) brought_scale[wave][q][lane / 16] = byte;
            }
        }
        if constexpr (RAW) {
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
            for (int q = 0; q < kAhead; ++q) {
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    wa[q][h] = *reinterpret_cast<const i32x4*>(&brought[wave][q][row % kRawRows * kBlock + at + 64 * h]);
                sa[q] = brought_scale[wave][q][row % kRawRows];
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        }
#pragma unroll
        for (int q = 0; q < kAhead; ++q) {
            if (kb0 + q * KS >= p.blocks) break;
            const i32x8 va = __builtin_shufflevector(wa[q][0], wa[q][1], 0, 1, 2, 3, 4, 5, 6, 7);
#pragma unroll
            for (int g = 0; g < NF; ++g) {
                const i32x8 vb = __builtin_shufflevector(wb[q][g][0], wb[q][g][1], 0, 1, 2, 3, 4, 5, 6, 7);
                if constexpr (WIDE) {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        acc[g] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                            to_bf16(vb[2 * e], vb[2 * e + 1], scale_of(sb[q][g])),
                            to_bf16(va[2 * e], va[2 * e + 1], scale_of(sa[q])), acc[g], 0, 0, 0);
                } else {
                    acc[g] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(vb, va, acc[g], 0, 0, 0, sb[q][g], 0, sa[q]);
                }
            }
            mfma_settle();  // (the next block is conditional)
        }
    }
    mfma_settle();
#pragma unroll
    for (int g = 0; g < NF; ++g) room[wave][g][lane] = acc[g];
    __syncthreads();
    if (wave >= NF) return;
    acc4 sum = room[0][wave][lane];
#pragma unroll
    for (int w = 1; w < KS; ++w) sum += room[w][wave][lane];
    store_four(p, row, j0 + 16 * wave + 4 * (lane / 16), sum, 0);
}

// Joins the parts of a split sum, in their order.
template <class O>
__global__ void __launch_bounds__(256) k_product_join(Product<O> p, int splits) {
    const i64 total = static_cast<i64>(p.m) * p.n;
    for (i64 e = static_cast<i64>(blockIdx.x) * 256 + threadIdx.x; e < total; e += static_cast<i64>(gridDim.x) * 256) {
        float sum = p.partial[e];
        for (int s = 1; s < splits; ++s) sum += p.partial[s * total + e];
        p.out[e / p.n * p.out_stride + e % p.n] = static_cast<O>(sum);
    }
}

template <class O>
__global__ void __launch_bounds__(256) k_product_zero(O* __restrict__ out, i64 out_stride, i64 m, i64 n) {
    for (i64 e = static_cast<i64>(blockIdx.x) * 256 + threadIdx.x; e < m * n; e += static_cast<i64>(gridDim.x) * 256)
        out[e / n * out_stride + e % n] = static_cast<O>(0.0f);
}

// How a product is cut: the tile, and parts of the summed axis.
struct Plan {
    int tile;    // 256, 128 or 64
    int groups;  // of waves that share a tile's blocks: 1, or 4 for few tiles of 64
    int splits;
    i64 split_blocks;
};

constexpr int kUnits = 256;  // compute units

// The tile is the one whose rounds over the card take least: a unit holds one tile of 256 at a
// time, two of 128 or four of 64, whose rates on large products are as 1 : 1/1.12 : 1/1.86 (2,600, 2,320 and
// 1,400 TFLOP/s at 8192 x 8192 x 8192), but one round of four tiles of 64 on every unit is slower than one of 128
// (2048 cubed 16.4 and 14.2 us).  20000 x 1024 x 512: 21.8 us in 316 tiles of 256, two rounds, 18.5 in 1,256 of 128.
// Four groups of waves share the blocks of a tile of 64 where that leaves no unit two of them and the sum is long enough
// for it: 1024 x 1024 x 2048 in 7.4 us (7.8 without), x 8192 in 20.9 (34.0), but x 512 in 5.0 (3.9).  Parts of the sum pay
// from 24 blocks on: 100 x 1000 x 4096 in 8.4 us in four parts (9.0), 512 x 1024 x 2048 in 9.8 us in two (6.8).
Plan plan_product(i64 m, i64 n, i64 k) {
    const auto tiles = [&](i64 t) { return (m + t - 1) / t * ((n + t - 1) / t); };
    const auto rounds = [&](i64 t, i64 held) { return (tiles(t) + held * kUnits - 1) / (held * kUnits); };
    const i64 blocks = (k + kBlock - 1) / kBlock;
    const bool full = tiles(64) > 3 * kUnits && tiles(64) <= 4 * kUnits;
    const double t256 = 1.0 * rounds(256, 1), t128 = 1.12 / 2 * rounds(128, 2), t64 = (full ? 2.4 : 1.86) / 4 * rounds(64, 4);
    Plan p{t256 <= t128 && t256 <= t64 ? 256 : t128 <= t64 ? 128 : 64, 1, 1, blocks};
    const i64 count = tiles(p.tile);
    if (p.tile == 64 && count <= kUnits && blocks >= 12) {
        p.groups = 4;
        // parts of at least eight blocks, up to a tile for each unit; a second launch joins them
        const i64 want = kUnits / count, most = blocks < 24 ? 1 : blocks / 8, parts = want < most ? want : most;
        if (parts > 1) {
            p.split_blocks = ((blocks + parts - 1) / parts + 3) / 4 * 4;  // scales are read four blocks at a time
            p.splits = static_cast<int>((blocks + p.split_blocks - 1) / p.split_blocks);
        }
    }
    return p;
}

i64 split_bytes(i64 m, i64 n, i64 k) {
    if (m <= kFewRows || n <= 0 || k <= 0) return 0;
    const Plan p = plan_product(m, n, k);
    return p.splits > 1 ? 4 * p.splits * m * n : 0;
}

// bytes of a matrix's blocks, scales included, as the workspace holds them
i64 block_bytes(i64 rows, i64 cols) { return rows * block_stride(cols) + (rows * block_scale_stride(cols) + 15) / 16 * 16; }

void check_sizes(i64 m, i64 n, i64 k) {
    constexpr i64 most = (1LL << 31) - 512;  // indexes of a tile past the end stay in 31 bits
    require(m >= 0 && m <= most && n >= 0 && n <= most && k >= 0 && k <= most, "sizes must be in [0, 2^31 - 512]");
}

// a tile of 256 rows is addressed with 31 bits
void check_summed(i64 k) {
    if (k > (1LL << 23) - kBlock) throw std::domain_error("products sum over up to 2^23 - 128 values");
}

void check_blocks(const void* values, const void* scales, i64 rows, i64 cols, const char* name) {
    if (rows == 0 || cols == 0) return;
    if (!values || !scales) throw std::invalid_argument(std::string(name) + " is NULL");
    if (!aligned(values, 16) || !aligned(scales, 16))
        throw std::invalid_argument(std::string(name) + ": 8-bit blocks must be 16-byte aligned");
}

template <class T>
void launch_quantize(const T* x, i64 x_stride, i64 rows, i64 cols, std::uint8_t* values, std::uint8_t* scales,
                     std::uint8_t* values_t, std::uint8_t* scales_t, hipStream_t stream) {
    const i64 pitch = block_stride(cols), scale_pitch = block_scale_stride(cols);
    if (!values_t) {
        const i64 groups = (rows * (pitch / kBlock) + 15) / 16;
        k_quantize_rows<T><<<static_cast<unsigned>(groups < 65536 ? groups : 65536), 256, 0, stream>>>(
            x, x_stride, rows, cols, values, scales, pitch, scale_pitch);
        SMX_LAUNCH_CHECK("k_quantize_rows");
        return;
    }
    const i64 tiles = block_stride(rows) / kBlock * (pitch / kBlock);
    require(tiles < (1LL << 31), "the matrix has too many tiles");
    (values ? k_quantize_tile<T, true> : k_quantize_tile<T, false>)<<<static_cast<unsigned>(tiles), 256, 0,
                                                                                stream>>>(
        x, x_stride, rows, cols, values, scales, pitch, scale_pitch, values_t, scales_t, block_stride(rows),
        block_scale_stride(rows));
    SMX_LAUNCH_CHECK("k_quantize_tile");
}

void quantize(const void* x, i64 x_stride, int dtype, i64 rows, i64 cols, std::uint8_t* values, std::uint8_t* scales,
              std::uint8_t* values_t, std::uint8_t* scales_t, hipStream_t stream) {
    if (rows == 0 || cols == 0 || (!values && !values_t)) return;
    with_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        launch_quantize(static_cast<const T*>(x), x_stride, rows, cols, values, scales, values_t, scales_t, stream);
    });
}

template <class O, bool WIDE>
void launch_tiles(const Product<O>& p, const Plan& plan, hipStream_t stream) {
    // as many workgroups as the card holds of a tile that goes on to the next, all otherwise
    const auto grid = [&](int held) {
        const int tiles = p.tiles_m * p.tiles_n, most = held * static_cast<int>(kUnits);
        return dim3(static_cast<unsigned>(tiles < most || held == 0 ? tiles : most), static_cast<unsigned>(plan.splits));
    };
    switch (plan.tile) {
        case 256: k_product_tile<O, WIDE, 256, 256, 2, 4, 1><<<grid(1), 512, 0, stream>>>(p); break;
        case 128: k_product_tile<O, WIDE, 128, 128, 2, 2, 1><<<grid(2), 256, 0, stream>>>(p); break;
        default:
            if (plan.groups == 1)
                k_product_tile<O, WIDE, 64, 64, 2, 2, 1><<<grid(4), 256, 0, stream>>>(p);
            else
                k_product_tile<O, WIDE, 64, 64, 2, 2, 4><<<grid(0), 1024, 0, stream>>>(p);
    }
    SMX_LAUNCH_CHECK("k_product_tile");
}

template <class T, class O, bool RAW>
void launch_rows(Product<O> p, const T* x, i64 x_stride, i64 k, hipStream_t stream) {
    const bool wide = sizeof(O) == 4 || k <= kShortSum;
    // 32 columns a workgroup where that is one for each unit, else 16
    const auto go = [&](auto w, auto nf) {
        constexpr int NF = decltype(nf)::value, KS = 8;
        k_product_rows<T, O, RAW, decltype(w)::value, NF, KS><<<blocks_for(p.n, 16 * NF), 64 * KS, 0, stream>>>(
            p, x, x_stride, static_cast<int>(k));
    };
    const auto with_form = [&](auto w) {
        using std::integral_constant;
        if (p.n >= 32 * kUnits)
            go(w, integral_constant<int, 2>{});
        else
            go(w, integral_constant<int, 1>{});
    };
    if (wide)
        with_form(std::true_type{});
    else
        with_form(std::false_type{});
    SMX_LAUNCH_CHECK("k_product_rows");
}

template <class O>
Product<O> product_of(const std::uint8_t* a, const std::uint8_t* as, const std::uint8_t* b, const std::uint8_t* bs, i64 m,
                      i64 n, i64 k, O* out, i64 out_stride) {
    Product<O> p{};
    p.a = a, p.as = as, p.b = b, p.bs = bs;
    p.m = static_cast<int>(m), p.n = static_cast<int>(n);
    p.blocks = static_cast<int>(block_stride(k) / kBlock);
    p.pitch = block_stride(k), p.scale_pitch = block_scale_stride(k);
    p.out = out, p.out_stride = out_stride;
    return p;
}

template <class O>
void launch_product(const std::uint8_t* a, const std::uint8_t* as, const std::uint8_t* b, const std::uint8_t* bs, i64 m,
                    i64 n, i64 k, O* out, i64 out_stride, float* partial, hipStream_t stream) {
    if (k == 0) {
        k_product_zero<O><<<static_cast<unsigned>(m * n < 256 * 4096 ? (m * n + 255) / 256 : 4096), 256, 0, stream>>>(
            out, out_stride, m, n);
        SMX_LAUNCH_CHECK("k_product_zero");
        return;
    }
    Product<O> p = product_of(a, as, b, bs, m, n, k, out, out_stride);
    if (m <= kFewRows) {
        launch_rows<O, O, false>(p, nullptr, 0, k, stream);
        return;
    }
    const Plan plan = plan_product(m, n, k);
    const i64 tiles_m = (m + plan.tile - 1) / plan.tile, tiles_n = (n + plan.tile - 1) / plan.tile;
    require(tiles_m * tiles_n < (1LL << 31) && 8 * tiles_n < (1LL << 31), "the product has too many tiles");
    p.partial = plan.splits > 1 ? partial : nullptr;
    p.split_blocks = static_cast<int>(plan.split_blocks);
    p.tiles_m = static_cast<int>(tiles_m), p.tiles_n = static_cast<int>(tiles_n);
    const bool wide = sizeof(O) == 4 || k <= kShortSum;
    (wide ? launch_tiles<O, true> : launch_tiles<O, false>)(p, plan, stream);
    if (plan.splits > 1) {
        k_product_join<O><<<static_cast<unsigned>(m * n < 256 * 4096 ? (m * n + 255) / 256 : 4096), 256, 0, stream>>>(
            p, plan.splits);
        SMX_LAUNCH_CHECK("k_product_join");
    }
}

}  // namespace
}  // namespace node
}  // namespace smx

using namespace smx;
using namespace smx::node;

extern "C" {

int64_t smx_block_stride(int64_t cols) { return cols > 0 ? block_stride(cols) : 0; }
int64_t smx_block_scale_stride(int64_t cols) { return cols > 0 ? block_scale_stride(cols) : 0; }

int32_t smx_block_quantize(const void* x, int64_t x_stride, int32_t dtype, int64_t rows, int64_t cols, uint8_t* values,
                           uint8_t* scales, uint8_t* values_t, uint8_t* scales_t, void* stream) {
    return guarded([&] {
        check_sizes(rows, cols, 0);
        require(dtype >= SMX_DTYPE_F32 && dtype <= SMX_DTYPE_F16, "unknown dtype code");
        check_rows(x, x_stride, rows, cols, dtype, "x");
        require(!values == !scales && !values_t == !scales_t, "values and scales go together");
        require(values || values_t || rows == 0 || cols == 0, "no output is asked for");
        if (values) check_blocks(values, scales, rows, cols, "values");
        if (values_t) check_blocks(values_t, scales_t, rows, cols, "values_t");
        quantize(x, x_stride, dtype, rows, cols, values, scales, values_t, scales_t, static_cast<hipStream_t>(stream));
    });
}

int64_t smx_block_product_workspace(int64_t m, int64_t n, int64_t k) { return split_bytes(m, n, k); }

int32_t smx_block_product(const uint8_t* a_values, const uint8_t* a_scales, const uint8_t* b_values,
                          const uint8_t* b_scales, int64_t m, int64_t n, int64_t k, int32_t dtype, void* out,
                          int64_t out_stride, void* workspace, int64_t workspace_bytes, void* stream) {
    return guarded([&] {
        check_sizes(m, n, k);
        require(dtype >= SMX_DTYPE_F32 && dtype <= SMX_DTYPE_F16, "unknown dtype code");
        check_blocks(a_values, a_scales, m, k, "a");
        check_blocks(b_values, b_scales, n, k, "b");
        check_rows(out, out_stride, m, n, dtype, "out");
        check_summed(k);
        check_workspace(workspace, workspace_bytes, smx_block_product_workspace(m, n, k));
        if (m == 0 || n == 0) return;
        with_dtype(dtype, [&](auto o) {
            using O = decltype(o);
            launch_product<O>(a_values, a_scales, b_values, b_scales, m, n, k, static_cast<O*>(out), out_stride,
                              static_cast<float*>(workspace), static_cast<hipStream_t>(stream));
        });
    });
}

int64_t smx_block_linear_workspace(int64_t m, int64_t n, int64_t k) {
    if (m <= kRawRows || n <= 0 || k <= 0) return 0;
    return block_bytes(m, k) + split_bytes(m, n, k);
}

int32_t smx_block_linear(const void* x, int64_t x_stride, int32_t dtype, const uint8_t* w_values,
                         const uint8_t* w_scales, int64_t m, int64_t n, int64_t k, int32_t out_dtype, void* out,
                         int64_t out_stride, void* workspace, int64_t workspace_bytes, void* stream) {
    return guarded([&] {
        check_sizes(m, n, k);
        require(dtype >= SMX_DTYPE_F32 && dtype <= SMX_DTYPE_F16, "unknown dtype code");
        require(out_dtype >= SMX_DTYPE_F32 && out_dtype <= SMX_DTYPE_F16, "unknown dtype code");
        check_rows(x, x_stride, m, k, dtype, "x");
        check_blocks(w_values, w_scales, n, k, "w");
        check_rows(out, out_stride, m, n, out_dtype, "out");
        check_summed(k);
        check_workspace(workspace, workspace_bytes, smx_block_linear_workspace(m, n, k));
        if (m == 0 || n == 0) return;
        if (m <= kRawRows && k > 0) {
            with_dtype(dtype, [&](auto t) {
                with_dtype(out_dtype, [&](auto o) {
                    using T = decltype(t);
                    using O = decltype(o);
                    launch_rows<T, O, true>(product_of<O>(nullptr, nullptr, w_values, w_scales, m, n, k, static_cast<O*>(out),
                                                          out_stride),
                                            static_cast<const T*>(x), x_stride, k, static_cast<hipStream_t>(stream));
                });
            });
            return;
        }
        auto* const values = static_cast<std::uint8_t*>(workspace);
        std::uint8_t* const scales = k > 0 ? values + m * block_stride(k) : nullptr;
        auto* const partial = k > 0 ? reinterpret_cast<float*>(values + block_bytes(m, k)) : nullptr;
        quantize(x, x_stride, dtype, m, k, values, scales, nullptr, nullptr, static_cast<hipStream_t>(stream));
        with_dtype(out_dtype, [&](auto o) {
            using O = decltype(o);
            launch_product<O>(values, scales, w_values, w_scales, m, n, k, static_cast<O*>(out), out_stride, partial,
                              static_cast<hipStream_t>(stream));
        });
    });
}

}  // extern "C"
