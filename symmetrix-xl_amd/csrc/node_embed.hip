// Species embedding: scaled rows of a table by type, and the gradient of the
// table, summed over the atoms of each type.
#include "node_ops.hpp"

namespace smx {
namespace node {
namespace {

// The type of atom t, or -1 where it is none of the table's.
template <class I>
__device__ __forceinline__ int type_of(const I* types, i64 t, i64 num_types) {
    const I z = types[t];
    return z >= 0 && static_cast<i64>(z) < num_types ? static_cast<int>(z) : -1;
}

// Lanes that share a row, eight channels each: a power of two up to a wave, which takes wider rows
// in slabs of 512.
inline int lanes_of(i64 channels, int most = 64) {
    int g = 8;
    while (g < most && 8 * g < channels) g *= 2;
    return g;
}

// A group of lanes a row: its type, then sixteen bytes a lane of the table's row and of out's.  Where out is more than the
// last cache holds (256 MB, the rows read included) a group has four rows, whose types are waited for together (a wait
// between the rows' loads would be for the rows before as well): 300,000 rows of 2 KB in 177 us, 212 at a row a group;
// 131,071 in 78 to 82, 82 to 98.  Below it one row: 65,536 rows of 1 KB in 20.8 us, 21.4 at four; 5,000 of 512 B, where
// latency counts, in 3.0 and 3.8.
constexpr i64 kManyBytes = i64{192} << 20;

template <class T, class I, int ROWS>
__global__ void __launch_bounds__(256) k_embed(const I* __restrict__ types, i64 tokens, const T* __restrict__ table,
                                               i64 table_stride, i64 num_types, int channels, float scale,
                                               T* __restrict__ out, i64 out_stride, int lanes) {
    const int groups = 256 / lanes;
    const int c = 8 * (blockIdx.y * lanes + threadIdx.x % lanes);
    if (c >= channels) return;
    for (i64 t0 = (static_cast<i64>(blockIdx.x) * groups + threadIdx.x / lanes) * ROWS; t0 < tokens;
         t0 += static_cast<i64>(gridDim.x) * groups * ROWS) {
        int z[ROWS];
        Eight<T> row[ROWS];
#pragma unroll
        for (int k = 0; k < ROWS; ++k) z[k] = type_of(types, t0 + k < tokens ? t0 + k : tokens - 1, num_types);
#pragma unroll
        for (int k = 0; k < ROWS; ++k) asm volatile("" : "+v"(z[k]));
#pragma unroll
        for (int k = 0; k < ROWS; ++k)
            if (z[k] >= 0) row[k] = load_pack(table + z[k] * table_stride, c, channels);
#pragma unroll
        for (int k = 0; k < ROWS; ++k) {
            if (t0 + k >= tokens) break;
            settle(row[k], c, channels);
            float v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = z[k] < 0 ? 0.0f : scale * row[k][i];
            store_eight(out + (t0 + k) * out_stride, c, channels, v);
        }
    }
}

// ---- the gradient of few atoms: no sort ----

// Up to kFew atoms, in one launch: a wave finds a row's atoms among 64 with a ballot and adds them up, its
// groups of lanes every so-manieth of them, joined between the lanes; rows without atoms get zeros.  WAVES > 1: a
// workgroup a row, 64 atoms a wave, joined in LDS; else, for many rows, a wave a row, all atoms.
// One launch in place of three: 135 atoms of 89 species x 32 15.0 -> 3.1 us, 256 atoms of one species x 1024, the
// slowest, 15.2.
constexpr int kFew = 256, kFewWide = 1024, kFewRows = 1024;

template <class T, class I, int WAVES>
__global__ void __launch_bounds__(WAVES > 1 ? 64 * WAVES : 256) k_embed_gradient_few(const I* __restrict__ types, int tokens,
                                                            const T* __restrict__ grad, i64 grad_stride, i64 num_types,
                                                            int channels, float scale, T* __restrict__ out, i64 out_stride,
                                                            int lanes) {
    constexpr bool WIDE = WAVES > 1;
    constexpr int kAhead = 8, kParts = WIDE ? 1 : kFew / 64;
    __shared__ float room[WAVES][WIDE ? 512 : 1];
    const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const int group = lane / lanes, groups = 64 / lanes, c0 = 8 * blockIdx.y * lanes, c = c0 + 8 * (lane % lanes);
    int mine[kParts];
#pragma unroll
    for (int k = 0; k < kParts; ++k) {
        const int t = 64 * (WIDE ? wave : k) + lane;
        mine[k] = t < tokens ? type_of(types, t, num_types) : -1;
    }
    for (i64 v = WIDE ? static_cast<i64>(blockIdx.x) : static_cast<i64>(blockIdx.x) * 4 + wave; v < num_types;
         v += static_cast<i64>(gridDim.x) * (WIDE ? 1 : 4)) {
        float sum[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int k = 0; k < kParts; ++k) {
            unsigned long long left = __ballot(mine[k] == static_cast<int>(v));
            while (left) {
                int atom[kAhead];
                Eight<T> row[kAhead];
#pragma unroll
                for (int j = 0; j < kAhead; ++j) {
                    atom[j] = -1;
                    for (int q = 0; q < groups && left; ++q, left &= left - 1)
                        if (q == group) atom[j] = 64 * (WIDE ? wave : k) + __builtin_ctzll(left);
                    if (atom[j] >= 0 && c < channels)
                        row[j] = load_pack(grad + static_cast<i64>(atom[j]) * grad_stride, c, channels);
                }
#pragma unroll
                for (int j = 0; j < kAhead; ++j)
                    if (atom[j] >= 0 && c < channels) {
                        settle(row[j], c, channels);
#pragma unroll
                        for (int i = 0; i < 8; ++i) sum[i] += row[j][i];
                    }
            }
        }
        for (int o = lanes; o < 64; o *= 2)
#pragma unroll
            for (int i = 0; i < 8; ++i) sum[i] += __shfl_xor(sum[i], o);
        if constexpr (WIDE) {
            if (group == 0)
#pragma unroll
                for (int i = 0; i < 8; ++i) room[wave][8 * lane + i] = sum[i];
            __syncthreads();
            for (int w = threadIdx.x; w < 8 * lanes && c0 + w < channels; w += 64 * WAVES) {
                float all = room[0][w];
#pragma unroll
                for (int k = 1; k < WAVES; ++k) all += room[k][w];
                out[v * out_stride + c0 + w] = static_cast<T>(scale * all);
            }
            __syncthreads();
        } else if (group == 0 && c < channels) {
#pragma unroll
            for (int i = 0; i < 8; ++i) sum[i] *= scale;
            store_eight(out + v * out_stride, c, channels, sum);
        }
    }
}

// ---- the gradient of few species: no sort ----

// The rows of the table in registers, V of them: a group of lanes, which hold a row, reads eight rows of the gradient
// at once (every groups-th of the workgroup's), and adds each to its type's; WAVE: a group is whole waves, whose
// rows' types are scalars (300,000 of 3 x 448 bf16: 77 us, 86 without).  The groups are joined in LDS, the workgroups' parts
// [blocks][num_types][channels] by k_embed_species_join, both in order.  One reading and two launches: 300,000 atoms of 3
// species x 448 FP32 in 106 us (5.1 TB/s; sorted 150), three waves a SIMD with eight rows under way each; 30,000 of 2 x
// 256 in 12.1 (23.9 sorted), where a round of rows is all there is.
template <class T, class I, int V, bool WAVE>
__global__ void __launch_bounds__(256, 3) k_embed_species(const I* __restrict__ types, i64 tokens, const T* __restrict__ grad,
                                                       i64 grad_stride, int num_types, int channels,
                                                       float* __restrict__ parts, int lanes, i64 chunk) {
    constexpr int kAhead = 8;
    __shared__ float room[256 * 8];
    const int groups = 256 / lanes, width = 8 * lanes, group = threadIdx.x / lanes, lane = threadIdx.x % lanes;
    const int c = 8 * lane;
    const i64 start = blockIdx.x * chunk, end = start + chunk < tokens ? start + chunk : tokens;
    float acc[V][8];
#pragma unroll
    for (int v = 0; v < V; ++v)
#pragma unroll
        for (int i = 0; i < 8; ++i) acc[v][i] = 0.0f;
    int next[kAhead];
    const auto read = [&](i64 t0) {
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            const i64 t = t0 + j * groups;
            next[j] = t < end ? type_of(types, t, num_types) : -1;
        }
    };
    read(start + group);
    for (i64 t0 = start + group; t0 < end; t0 += kAhead * groups) {
        int z[kAhead];
        Eight<T> row[kAhead];
#pragma unroll
        for (int j = 0; j < kAhead; ++j) asm volatile("" : "+v"(next[j]));  // waited for together, before the rows' loads
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            z[j] = WAVE ? __builtin_amdgcn_readfirstlane(next[j]) : next[j];
            if (z[j] >= 0 && c < channels) row[j] = load_pack(grad + (t0 + j * groups) * grad_stride, c, channels);
        }
        read(t0 + kAhead * groups);
        settle(row, c, channels);
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
#pragma unroll
            for (int v = 0; v < V; ++v)
                if (z[j] == v)
#pragma unroll
                    for (int i = 0; i < 8; ++i) acc[v][i] += row[j][i];
        }
    }
#pragma unroll
    for (int v = 0; v < V; ++v) {
        if (v >= num_types) break;
#pragma unroll
        for (int i = 0; i < 8; ++i) room[group * width + 8 * lane + i] = acc[v][i];
        __syncthreads();
        for (int w = threadIdx.x; w < channels; w += 256) {
            float sum = room[w];
            for (int g = 1; g < groups; ++g) sum += room[g * width + w];
            parts[(static_cast<i64>(blockIdx.x) * num_types + v) * channels + w] = sum;
        }
        __syncthreads();
    }
}

template <class T>
__global__ void __launch_bounds__(1024) k_embed_species_join(const float* __restrict__ parts, int count, int num_types,
                                                             int channels, float scale, T* __restrict__ out, i64 out_stride) {
    const i64 size = static_cast<i64>(num_types) * channels;
    const i64 at = static_cast<i64>(blockIdx.x) * kJoined + threadIdx.x % kJoined;
    const float sum = sum_of_parts(parts + at, size, count, at < size);
    if (threadIdx.x >= kJoined || at >= size) return;
    out[at / channels * out_stride + at % channels] = static_cast<T>(scale * sum);
}

// ---- the gradient: atoms sorted by type, then runs of one type added up ----
//
// The sort is a stable radix sort of (type, atom), eight bits a pass, least first; types outside the
// table sort last as num_types.  Up to kSmall atoms one workgroup sorts in LDS; above, tiles of
// kTile atoms (times up to 512 tiles) are counted, and each pass places a tile's atoms by the counts of all tiles
// before it.  The sort is latency, not bytes: 5 us a pass in one workgroup, 3.8 + 6.8 for 30,000 atoms.

constexpr int kUnits = 256;  // compute units
constexpr int kDigits = 256, kTile = 1024, kMostTiles = 512, kSmall = 4096;

// the lanes of the wave that are `in` and hold the same digit
__device__ __forceinline__ unsigned long long same_digit(int digit, bool in) {
    unsigned long long m = __ballot(in);
#pragma unroll
    for (int b = 0; b < 8; ++b) {
        const bool one = digit >> b & 1;
        const unsigned long long w = __ballot(one);
        m &= one ? w : ~w;
    }
    return m;
}

// What a workgroup of WAVES waves ranks its atoms with.
template <int WAVES>
struct RankRoom {
    int count[WAVES][kDigits];  // of each wave, then the place of each wave's first
    int total[kDigits];
    int wave_total[4];
};

// Exclusive sums over the 256 digits: thread d < 256 gives its value and gets the sum of those before it.
// Every thread of the workgroup calls it.
template <int WAVES>
__device__ __forceinline__ int digits_before(int v, RankRoom<WAVES>& room) {
    const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
    int sum = v;
#pragma unroll
    for (int o = 1; o < 64; o *= 2) {
        const int below = __shfl_up(sum, o);
        if (lane >= o) sum += below;
    }
    if (threadIdx.x < kDigits && lane == 63) room.wave_total[wave] = sum;
    __syncthreads();
    int before = sum - v;
    for (int w = 0; w < wave && w < 4; ++w) before += room.wave_total[w];
    __syncthreads();
    return before;
}

// Ranks N atoms a lane (64 neighbouring ones a round, a wave's rounds neighbouring): rank[k] among the wave's
// atoms of the same digit, the waves' counts in room.count.
template <int WAVES, int N>
__device__ __forceinline__ void rank_in_wave(const int (&digit)[N], const bool (&in)[N], int (&rank)[N],
                                             RankRoom<WAVES>& room) {
    const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
    for (int d = lane; d < kDigits; d += 64) room.count[wave][d] = 0;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < N; ++k) {
        const unsigned long long same = same_digit(digit[k], in[k]);
        const int before = __popcll(same & ((1ull << lane) - 1));
        const int had = in[k] ? room.count[wave][digit[k]] : 0;
        rank[k] = had + before;
        __builtin_amdgcn_wave_barrier();
        if (in[k] && before == 0) room.count[wave][digit[k]] = had + __popcll(same);
        __builtin_amdgcn_wave_barrier();
    }
    __syncthreads();
}

template <class I>
__device__ __forceinline__ int sort_key(const I* types, i64 t, i64 num_types) {
    const int z = type_of(types, t, num_types);
    return z < 0 ? static_cast<int>(num_types) : z;
}

// One workgroup sorts up to kSmall atoms; the others clear `seen`.
template <class I>
__global__ void __launch_bounds__(1024) k_sort_small(const I* __restrict__ types, int tokens, i64 num_types, int bits,
                                                     int* __restrict__ keys, int* __restrict__ order,
                                                     std::uint8_t* __restrict__ seen) {
    constexpr int kWaves = 16, N = kSmall / 1024;
    __shared__ RankRoom<kWaves> room;
    __shared__ int skey[kSmall], satom[kSmall];
    if (blockIdx.x > 0) {
        for (i64 v = static_cast<i64>(blockIdx.x - 1) * 1024 + threadIdx.x; v < num_types;
             v += static_cast<i64>(gridDim.x - 1) * 1024)
            seen[v] = 0;
        return;
    }
    const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
    int key[N], atom[N], digit[N], rank[N];
    bool in[N];
#pragma unroll
    for (int k = 0; k < N; ++k) {
        atom[k] = wave * 64 * N + 64 * k + lane;
        in[k] = atom[k] < tokens;
        key[k] = in[k] ? sort_key(types, atom[k], num_types) : 0;
    }
    for (int shift = 0; shift < bits; shift += 8) {
#pragma unroll
        for (int k = 0; k < N; ++k) digit[k] = key[k] >> shift & (kDigits - 1);
        rank_in_wave<kWaves, N>(digit, in, rank, room);
        int total = 0;
        if (threadIdx.x < kDigits)
            for (int w = 0; w < kWaves; ++w) total += room.count[w][threadIdx.x];
        int place = digits_before<kWaves>(threadIdx.x < kDigits ? total : 0, room);
        if (threadIdx.x < kDigits)
            for (int w = 0; w < kWaves; ++w) {
                const int n = room.count[w][threadIdx.x];
                room.count[w][threadIdx.x] = place;
                place += n;
            }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < N; ++k)
            if (in[k]) {
                const int to = room.count[wave][digit[k]] + rank[k];
                skey[to] = key[k];
                satom[to] = atom[k];
            }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < N; ++k) {
            const int p = wave * 64 * N + 64 * k + lane;
            if (in[k]) key[k] = skey[p], atom[k] = satom[p];  // (in[k] is that of the place as well)
        }
        __syncthreads();
    }
#pragma unroll
    for (int k = 0; k < N; ++k)
        if (in[k]) keys[wave * 64 * N + 64 * k + lane] = key[k], order[wave * 64 * N + 64 * k + lane] = atom[k];
}

// Counts a pass's digits of each tile, of the types or of the pass before's keys, into counts [tiles][256]; clears
// `seen` where it is given.  (Counted by each pass for the next as it places its atoms, with atomics across the card, the
// sort of 300,000 atoms took 44 us more.)
template <class I>
__global__ void __launch_bounds__(256) k_sort_count(const I* __restrict__ types, i64 tokens, i64 num_types, int tile,
                                                    int shift, int* __restrict__ counts, std::uint8_t* __restrict__ seen) {
    __shared__ int count[kDigits];
    count[threadIdx.x] = 0;
    __syncthreads();
    const i64 first = static_cast<i64>(blockIdx.x) * tile, last = first + tile < tokens ? first + tile : tokens;
    for (i64 t = first + threadIdx.x; t < last; t += 256)
        atomicAdd(&count[sort_key(types, t, num_types) >> shift & (kDigits - 1)], 1);
    __syncthreads();
    const i64 hop = static_cast<i64>(gridDim.x) * 256, me = static_cast<i64>(blockIdx.x) * 256 + threadIdx.x;
    counts[me] = count[threadIdx.x];
    if (!seen) return;
    for (i64 v = me; v < num_types; v += hop) seen[v] = 0;
}

// One pass: a tile's atoms to their places, sixteen waves a workgroup (a pass is latency: its reads of the
// counts, its scan and its scattered stores).  counts: this pass's [tiles][256].  The first pass (types
// given) reads the types themselves.
template <class I>
__global__ void __launch_bounds__(1024) k_sort_place(const I* __restrict__ types, const int* __restrict__ keys_in,
                                                     const int* __restrict__ order_in, i64 tokens, i64 num_types, int tile,
                                                     int shift, const int* __restrict__ counts,
                                                     int* __restrict__ keys, int* __restrict__ order) {
    constexpr int kWaves = 16, N = kTile / 1024;
    __shared__ RankRoom<kWaves> room;
    __shared__ int base[kDigits], part[2][4][kDigits];
    const int lane = threadIdx.x % 64, wave = threadIdx.x / 64, mine = threadIdx.x % kDigits, quarter = threadIdx.x / kDigits;
    int before = 0, total = 0;
#pragma unroll 8
    for (int b = quarter; b < static_cast<int>(gridDim.x); b += 4) {
        const int n = counts[b * kDigits + mine];
        before += b < static_cast<int>(blockIdx.x) ? n : 0;
        total += n;
    }
    part[0][quarter][mine] = before;
    part[1][quarter][mine] = total;
    __syncthreads();
    before = part[0][0][mine] + part[0][1][mine] + part[0][2][mine] + part[0][3][mine];
    total = part[1][0][mine] + part[1][1][mine] + part[1][2][mine] + part[1][3][mine];
    const int start = digits_before<kWaves>(total, room) + before;
    if (threadIdx.x < kDigits) base[mine] = start;
    const i64 first = static_cast<i64>(blockIdx.x) * tile, last = first + tile < tokens ? first + tile : tokens;
    for (i64 at = first; at < last; at += kTile) {
        int key[N], atom[N], digit[N], rank[N];
        bool in[N];
#pragma unroll
        for (int k = 0; k < N; ++k) {
            const i64 p = at + wave * 64 * N + 64 * k + lane;
            in[k] = p < last;
            key[k] = !in[k] ? 0 : types ? sort_key(types, p, num_types) : keys_in[p];
            atom[k] = !in[k] ? 0 : types ? static_cast<int>(p) : order_in[p];
            digit[k] = key[k] >> shift & (kDigits - 1);
        }
        rank_in_wave<kWaves, N>(digit, in, rank, room);
        if (threadIdx.x < kDigits) {
            int place = base[mine];
            for (int w = 0; w < kWaves; ++w) {
                const int n = room.count[w][mine];
                room.count[w][mine] = place;
                place += n;
            }
            base[mine] = place;
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < N; ++k)
            if (in[k]) {
                const int to = room.count[wave][digit[k]] + rank[k];
                keys[to] = key[k];
                order[to] = atom[k];
            }
        __syncthreads();
    }
}

// Sorted atoms that a group of lanes adds up: as many, with as few parts to join, as still fill the
// card (300,000 atoms of 5 species x 447: 214 us at 16, 171 at 64).
constexpr int kRuns[3] = {64, 16, 8};

// 256 / lanes groups a workgroup, each `length` sorted atoms of 8 lanes' channels.  A type whose atoms lie
// within a group is done there; the first and last runs of the groups are joined in LDS, in order; what crosses
// the workgroup's ends leaves as a part: [0] of a run that goes on from the workgroup before, [1] of one that starts here
// and goes on in the next.  Bound by the gathered rows: 131,071 of 2 KB in 76 us (3.5 TB/s, and 0.7 of stores), eight
// of them under way a group and the next eight's places read meanwhile.  WHOLE: rows of whole eights of channels, whose
// loads have no ends to settle (300,000 of 448 FP32 153 us, 173 with them; of 447 176).
template <class T, bool WHOLE>
__global__ void __launch_bounds__(256) k_embed_runs(const int* __restrict__ keys, const int* __restrict__ order, i64 tokens,
                                                    const T* __restrict__ grad, i64 grad_stride, int num_types,
                                                    int channels, float scale, T* __restrict__ out, i64 out_stride,
                                                    float* __restrict__ parts, std::uint8_t* __restrict__ seen, int lanes, int length) {
    __shared__ int piece_key[2 * 32];
    __shared__ float piece[2 * 256 * 8];
    const int groups = 256 / lanes, width = 8 * lanes, group = threadIdx.x / lanes, lane = threadIdx.x % lanes;
    const int c0 = blockIdx.y * width, c = c0 + 8 * lane;
    const i64 chunk = static_cast<i64>(groups) * length, start = blockIdx.x * chunk;
    const i64 end = start + chunk < tokens ? start + chunk : tokens;
    const i64 first = start + group * length;
    float acc[8], head[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) acc[i] = head[i] = 0.0f;
    int current = -1, head_key = -1;  // no run yet
    bool in_head = true;
    const auto close = [&]() {
        if (in_head) {
            head_key = current;
#pragma unroll
            for (int i = 0; i < 8; ++i) head[i] = acc[i];
            in_head = false;
        } else if (c < channels) {
            float v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = scale * acc[i];
            store_eight(out + static_cast<i64>(current) * out_stride, c, channels, v);
        }
        if (lane == 0 && blockIdx.y == 0) seen[current] = 1;
#pragma unroll
        for (int i = 0; i < 8; ++i) acc[i] = 0.0f;
    };
    const int before = start > 0 ? keys[start - 1] : -1, after = end < tokens ? keys[end] : num_types;
    int key[8], atom[8];
    const auto read = [&](int b) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const i64 p = first + b + j < end ? first + b + j : end - 1;
            key[j] = first + b + j < end ? keys[p] : num_types;
            atom[j] = order[p];
        }
    };
    read(0);
    for (int b = 0; b < length; b += 8) {
        int here[8];
        Eight<T> row[8];
        // all eight places are waited for here: a wait between the rows' loads would be for the rows before as well
        // (131,071 rows of 2 KB: 84 -> 76 us)
#pragma unroll
        for (int j = 0; j < 8; ++j) asm volatile("" : "+v"(key[j]), "+v"(atom[j]));
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            here[j] = key[j];
            if (here[j] < num_types && c < channels)
                row[j] = load_pack(grad + static_cast<i64>(atom[j]) * grad_stride, c, WHOLE ? c + 8 : channels);
        }
        if (b + 8 < length) read(b + 8);
        if constexpr (!WHOLE) settle(row, c, channels);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            if (here[j] >= num_types) continue;  // past the end, or no species: these sort last
            if (here[j] != current) {
                if (current >= 0) close();
                current = here[j];
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) acc[i] += row[j][i];
        }
    }
    // a group's pieces: its first run and, where it has another, its last
    const bool one = in_head;
    if (lane == 0) {
        piece_key[2 * group] = one ? current : head_key;
        piece_key[2 * group + 1] = one ? -1 : current;
        if (current >= 0 && blockIdx.y == 0) seen[current] = 1;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        piece[2 * group * width + 8 * lane + i] = one ? acc[i] : head[i];
        piece[(2 * group + 1) * width + 8 * lane + i] = acc[i];
    }
    __syncthreads();
    for (int w = threadIdx.x; w < width && c0 + w < channels; w += 256) {
        float sum = 0.0f;
        int run = -1;
        bool from_before = false;
        for (int q0 = 0; q0 < 2 * groups; q0 += 8) {  // (at least four groups)
            int next[8];
            float value[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) next[j] = piece_key[q0 + j], value[j] = piece[(q0 + j) * width + w];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                if (next[j] < 0) continue;
                if (next[j] != run) {
                    if (run >= 0) {
                        if (from_before)
                            parts[(2 * static_cast<i64>(blockIdx.x)) * channels + c0 + w] = sum;
                        else
                            out[run * out_stride + c0 + w] = static_cast<T>(scale * sum);
                    }
                    from_before = run < 0 && next[j] == before;
                    run = next[j];
                    sum = 0.0f;
                }
                sum += value[j];
            }
        }
        if (run < 0) continue;
        if (from_before)
            parts[(2 * static_cast<i64>(blockIdx.x)) * channels + c0 + w] = sum;
        else if (run == after)
            parts[(2 * static_cast<i64>(blockIdx.x) + 1) * channels + c0 + w] = sum;
        else
            out[run * out_stride + c0 + w] = static_cast<T>(scale * sum);
    }
}

// Zeros for the types without atoms (workgroups from `chunks` on, a wave a row), and the joins of runs
// that cross workgroups: workgroup b's, if a run starts in b's atoms and goes on.  A run of few parts is
// added up by a thread a channel; one of many (thousands of atoms of a species) by eight waves, four channels
// a lane, an eighth of the parts each.
template <class T>
__global__ void __launch_bounds__(512) k_embed_finish(const int* __restrict__ keys, i64 tokens, int num_types, int channels,
                                                       float scale, T* __restrict__ out, i64 out_stride,
                                                       const float* __restrict__ parts,
                                                       const std::uint8_t* __restrict__ seen, i64 chunk, int chunks) {
    constexpr int kWaves = 8;
    __shared__ Pack<float, 4> room[kWaves][64];
    const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
    if (static_cast<int>(blockIdx.x) >= chunks) {
        const i64 hop = (static_cast<i64>(gridDim.x) - chunks) * kWaves;
        for (i64 v = (static_cast<i64>(blockIdx.x) - chunks) * kWaves + wave; v < num_types; v += hop) {
            if (seen[v]) continue;
            const float zeros[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
            for (int c = 8 * lane; c < channels; c += 512) store_eight(out + v * out_stride, c, channels, zeros);
        }
        return;
    }
    const i64 start = blockIdx.x * chunk, end = start + chunk;
    if (end >= tokens) return;
    const int run = keys[end - 1];
    if (run >= num_types || keys[end] != run) return;
    if (keys[start] == run && start > 0 && keys[start - 1] == run) return;  // it started before
    // the first place past the run: the 64 lanes narrow the range down together
    i64 low = end, high = tokens;
    while (high - low > 1) {  // keys[low] == run, and keys[high] != run where it exists
        const i64 hop = (high - low + 63) / 64, p = low + (lane + 1) * hop;
        const int same = __popcll(__ballot(p < high && keys[p] == run));
        const i64 up = low + (same + 1) * hop;
        low += same * hop;
        high = up < high ? up : high;
    }
    const i64 last = low / chunk;  // the workgroup of the run's last atom
    const float* const mine = parts + (2 * static_cast<i64>(blockIdx.x) + 1) * channels;
    const i64 hop = 2LL * channels;
    if (last - blockIdx.x <= 2 * kWaves) {
        for (int c = threadIdx.x; c < channels; c += 512) {
            float sum = mine[c];
            const float* at = parts + (static_cast<i64>(blockIdx.x) + 1) * hop + c;
            for (i64 b = blockIdx.x + 1; b <= last; ++b, at += hop) sum += *at;
            out[run * out_stride + c] = static_cast<T>(scale * sum);
        }
        return;
    }
    for (int c0 = 0; c0 < channels; c0 += 256) {
        const int c = c0 + 4 * lane;
        float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        const auto add = [&](const float* part) {
            if (c + 4 <= channels) {
                const Pack<float, 4> v = *reinterpret_cast<const Pack<float, 4>*>(part + c);
#pragma unroll
                for (int i = 0; i < 4; ++i) sum[i] += v.v[i];
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) sum[i] += c + i < channels ? part[c + i] : 0.0f;
            }
        };
        if (wave == 0) add(mine);
#pragma unroll 8
        for (i64 b = blockIdx.x + 1 + wave; b <= last; b += kWaves) add(parts + b * hop);
#pragma unroll
        for (int i = 0; i < 4; ++i) room[wave][lane].v[i] = sum[i];
        __syncthreads();
        if (threadIdx.x < 256 && c0 + static_cast<int>(threadIdx.x) < channels) {
            float s = 0.0f;
#pragma unroll
            for (int w = 0; w < kWaves; ++w) s += room[w][threadIdx.x / 4].v[threadIdx.x % 4];
            out[run * out_stride + c0 + threadIdx.x] = static_cast<T>(scale * s);
        }
        __syncthreads();
    }
}

// More than kFew only where a wave adds several rows at once: 1,000 atoms of 89 species x 128 take 3.5 us so and 14.9
// sorted, of one species 12.6 and 14.3, but of one species x 512 42 and 16.
bool few_atoms(i64 tokens, i64 num_types, i64 channels) {
    return tokens <= (num_types <= kFewRows && channels <= 256 ? kFewWide : kFew);
}

// Up to four species, whose rows the registers hold (eight take two waves a SIMD: 300,000 atoms x 448 bf16 101 us, 80
// sorted), in rows of up to a workgroup's channels (100,000 atoms x 4,096 bf16 in two slabs 266 us, 218 sorted), where a type
// has enough atoms for it: 1,000 atoms x 128 of one species 6.8 us, 12.7 in one launch; of three 9.5 and 6.3.
constexpr i64 kSpecies = 4;
constexpr int kSpeciesLanes = 256;

bool few_species(i64 tokens, i64 num_types, i64 channels) {
    return num_types <= kSpecies && channels <= 8 * kSpeciesLanes &&
           tokens > (few_atoms(tokens, num_types, channels) ? 2 * kFew * num_types : kFew);
}

// The three workgroups that a unit holds, or as many as take whole rounds of rows (30,000 atoms of 4 x 1,024 FP32:
// 38.7 us, 31.6 in whole rounds), and parts of at most an eighth of the rows.
i64 species_blocks(i64 tokens, i64 num_types, i64 channels) {
    const int lanes = lanes_of(channels, kSpeciesLanes);
    const i64 round = 8 * (256 / lanes), rounds = (tokens + round - 1) / round, most = tokens / (8 * num_types);
    const i64 each = (rounds + 3 * kUnits - 1) / (3 * kUnits), blocks = (rounds + each - 1) / each;
    return blocks < most ? blocks : most;
}

// The parts of a gradient call's workspace, in bytes from its start.
struct Workspace {
    i64 keys[2], order[2], counts, seen, parts, size;
    int passes, tile, tiles, lanes, length, chunks;
    i64 chunk;
};

Workspace plan_gradient(i64 tokens, i64 num_types, i64 channels) {
    Workspace w{};
    int bits = 1;
    while (num_types >> bits) ++bits;  // keys run to num_types
    w.passes = (bits + 7) / 8;
    w.tile = kTile * static_cast<int>((tokens + static_cast<i64>(kTile) * kMostTiles - 1) / (static_cast<i64>(kTile) * kMostTiles));
    if (w.tile == 0) w.tile = kTile;
    w.tiles = static_cast<int>((tokens + w.tile - 1) / w.tile);
    w.lanes = lanes_of(channels);
    const i64 groups = 256 / w.lanes;
    for (const int run : kRuns) {
        w.length = run;
        if (tokens >= groups * run * kUnits) break;
    }
    w.chunk = groups * w.length;
    w.chunks = static_cast<int>((tokens + w.chunk - 1) / w.chunk);
    const auto take = [&](i64 bytes) {
        const i64 at = w.size;
        w.size += (bytes + 15) / 16 * 16;
        return at;
    };
    const bool small = tokens <= kSmall;
    w.keys[0] = take(4 * tokens);
    w.order[0] = take(4 * tokens);
    if (!small) {
        w.keys[1] = take(4 * tokens);
        w.order[1] = take(4 * tokens);
        w.counts = take(4LL * kDigits * w.tiles);
    }
    w.seen = take(num_types);
    w.parts = take(8LL * w.chunks * channels);
    return w;
}

template <class F>
void with_index(int32_t wide, F&& f) {
    if (wide)
        f(std::int64_t{});
    else
        f(std::int32_t{});
}

void check_embed(const void* types, int32_t wide, i64 tokens, i64 num_types, i64 channels, int dtype) {
    constexpr i64 most = (1LL << 31) - 65536;  // indexes of a tile past the end stay in 31 bits
    require(tokens >= 0 && tokens <= most, "tokens must be in [0, 2^31 - 65536]");
    require(num_types >= 0 && num_types <= most, "num_types must be in [0, 2^31 - 65536]");
    require(channels >= 0 && channels <= 65535 * 512, "channels must be in [0, 65535 * 512]");
    require(dtype >= SMX_DTYPE_F32 && dtype <= SMX_DTYPE_F16, "unknown dtype code");
    require(tokens == 0 || types, "types is NULL");
    require(aligned(types, wide ? 8 : 4), "types is not aligned to its values");
}

}  // namespace
}  // namespace node
}  // namespace smx

using namespace smx;
using namespace smx::node;

extern "C" {

int32_t smx_embed(const void* types, int32_t types_are_64bit, int64_t tokens, const void* table, int64_t table_stride,
                  int64_t num_types, int64_t channels, int32_t dtype, float scale, void* out, int64_t out_stride,
                  void* stream) {
    return guarded([&] {
        check_embed(types, types_are_64bit, tokens, num_types, channels, dtype);
        check_rows(table, table_stride, num_types, channels, dtype, "table");
        check_rows(out, out_stride, tokens, channels, dtype, "out");
        if (tokens == 0 || channels == 0) return;
        with_dtype(dtype, [&](auto t) {
            using T = decltype(t);
            with_index(types_are_64bit, [&](auto i) {
                using I = decltype(i);
                const bool many = tokens * channels * static_cast<i64>(sizeof(T)) >= kManyBytes;
                const int lanes = lanes_of(channels), rows = 256 / lanes * (many ? 4 : 1);
                const i64 want = (tokens + rows - 1) / rows;
                (many ? k_embed<T, I, 4> : k_embed<T, I, 1>)<<<
                    dim3(static_cast<unsigned>(want < (1 << 20) ? want : 1 << 20), blocks_for(channels, 8 * lanes)), 256, 0,
                    static_cast<hipStream_t>(stream)>>>(static_cast<const I*>(types), tokens, static_cast<const T*>(table),
                                                        table_stride, num_types, static_cast<int>(channels), scale,
                                                        static_cast<T*>(out), out_stride, lanes);
                SMX_LAUNCH_CHECK("k_embed");
            });
        });
    });
}

int64_t smx_embed_gradient_workspace(int64_t tokens, int64_t num_types, int64_t channels) {
    if (num_types <= 0 || channels <= 0) return 0;
    if (few_species(tokens, num_types, channels)) return 4 * species_blocks(tokens, num_types, channels) * num_types * channels;
    if (few_atoms(tokens, num_types, channels)) return 0;
    return plan_gradient(tokens, num_types, channels).size;
}

int32_t smx_embed_gradient(const void* types, int32_t types_are_64bit, int64_t tokens, const void* grad,
                           int64_t grad_stride, int64_t num_types, int64_t channels, int32_t dtype, float scale,
                           void* out, int64_t out_stride, void* workspace, int64_t workspace_bytes, void* stream) {
    return guarded([&] {
        check_embed(types, types_are_64bit, tokens, num_types, channels, dtype);
        check_rows(grad, grad_stride, tokens, channels, dtype, "grad");
        check_rows(out, out_stride, num_types, channels, dtype, "out");
        check_workspace(workspace, workspace_bytes, smx_embed_gradient_workspace(tokens, num_types, channels));
        if (num_types == 0 || channels == 0) return;
        const auto queue = static_cast<hipStream_t>(stream);
        if (few_species(tokens, num_types, channels)) {
            const int lanes = lanes_of(channels, kSpeciesLanes), v = static_cast<int>(num_types), c = static_cast<int>(channels);
            const i64 blocks = species_blocks(tokens, num_types, channels), chunk = (tokens + blocks - 1) / blocks;
            auto* const parts = static_cast<float*>(workspace);
            with_dtype(dtype, [&](auto t) {
                using T = decltype(t);
                with_index(types_are_64bit, [&](auto i) {
                    using I = decltype(i);
                    (lanes >= 64 ? v <= 2 ? k_embed_species<T, I, 2, true> : k_embed_species<T, I, kSpecies, true>
                     : v <= 2    ? k_embed_species<T, I, 2, false>
                                 : k_embed_species<T, I, kSpecies, false>)<<<
                        static_cast<unsigned>(blocks), 256, 0, queue>>>(
                        static_cast<const I*>(types), tokens, static_cast<const T*>(grad), grad_stride, v, c, parts, lanes,
                        chunk);
                });
                SMX_LAUNCH_CHECK("k_embed_species");
                k_embed_species_join<T><<<blocks_for(num_types * channels, kJoined), 1024, 0, queue>>>(
                    parts, static_cast<int>(blocks), v, c, scale, static_cast<T*>(out), out_stride);
                SMX_LAUNCH_CHECK("k_embed_species_join");
            });
            return;
        }
        if (few_atoms(tokens, num_types, channels)) {
            const int lanes = lanes_of(channels), waves = num_types > kFewRows ? 1 : tokens <= kFew ? kFew / 64 : kFewWide / 64;
            const unsigned rows = waves > 1 ? static_cast<unsigned>(num_types) : blocks_for(num_types, 4);
            with_dtype(dtype, [&](auto t) {
                using T = decltype(t);
                with_index(types_are_64bit, [&](auto i) {
                    using I = decltype(i);
                    (waves == 1   ? k_embed_gradient_few<T, I, 1>
                     : waves == 4 ? k_embed_gradient_few<T, I, kFew / 64>
                                  : k_embed_gradient_few<T, I, kFewWide / 64>)<<<
                        dim3(rows < 4096 ? rows : 4096, blocks_for(channels, 8 * lanes)), waves > 1 ? 64 * waves : 256, 0,
                        queue>>>(static_cast<const I*>(types), static_cast<int>(tokens), static_cast<const T*>(grad),
                                 grad_stride, num_types, static_cast<int>(channels), scale, static_cast<T*>(out), out_stride,
                                 lanes);
                });
            });
            SMX_LAUNCH_CHECK("k_embed_gradient_few");
            return;
        }
        const Workspace w = plan_gradient(tokens, num_types, channels);
        auto* const base = static_cast<std::uint8_t*>(workspace);
        const auto ints = [&](i64 at) { return reinterpret_cast<int*>(base + at); };
        std::uint8_t* const seen = base + w.seen;
        int at = 0;  // which of the two buffers holds the sorted atoms
        with_index(types_are_64bit, [&](auto i) {
            using I = decltype(i);
            const I* const z = static_cast<const I*>(types);
            if (tokens <= kSmall) {
                const unsigned clear = blocks_for(num_types, 16 * 1024);
                k_sort_small<I><<<1 + (clear < 255 ? clear : 255), 1024, 0, queue>>>(
                    z, static_cast<int>(tokens), num_types, 8 * w.passes, ints(w.keys[0]), ints(w.order[0]), seen);
                SMX_LAUNCH_CHECK("k_sort_small");
                return;
            }
            for (int p = 0; p < w.passes; ++p, at ^= 1) {
                int* const counts = ints(w.counts);
                if (p == 0)
                    k_sort_count<I><<<w.tiles, 256, 0, queue>>>(z, tokens, num_types, w.tile, 0, counts, seen);
                else
                    k_sort_count<int><<<w.tiles, 256, 0, queue>>>(ints(w.keys[at ^ 1]), tokens, num_types, w.tile, 8 * p, counts,
                                                                  nullptr);
                SMX_LAUNCH_CHECK("k_sort_count");
                k_sort_place<I><<<w.tiles, 1024, 0, queue>>>(p ? nullptr : z, ints(w.keys[at ^ 1]), ints(w.order[at ^ 1]), tokens,
                                                             num_types, w.tile, 8 * p, counts, ints(w.keys[at]),
                                                             ints(w.order[at]));
                SMX_LAUNCH_CHECK("k_sort_place");
            }
            at ^= 1;
        });
        with_dtype(dtype, [&](auto t) {
            using T = decltype(t);
            auto* const parts = reinterpret_cast<float*>(base + w.parts);
            if (tokens > 0) {
                (channels % 8 == 0 ? k_embed_runs<T, true> : k_embed_runs<T, false>)<<<dim3(static_cast<unsigned>(w.chunks), blocks_for(channels, 8 * w.lanes)), 256, 0, queue>>>(
                    ints(w.keys[at]), ints(w.order[at]), tokens, static_cast<const T*>(grad), grad_stride,
                    static_cast<int>(num_types), static_cast<int>(channels), scale, static_cast<T*>(out), out_stride, parts,
                    seen, w.lanes, w.length);
                SMX_LAUNCH_CHECK("k_embed_runs");
            }
            const unsigned rows = blocks_for(num_types, 8);
            k_embed_finish<T><<<static_cast<unsigned>(w.chunks) + (rows < 4096 ? rows : 4096), 512, 0, queue>>>(
                ints(w.keys[at]), tokens, static_cast<int>(num_types), static_cast<int>(channels), scale,
                static_cast<T*>(out), out_stride, parts, seen, w.chunk, w.chunks);
            SMX_LAUNCH_CHECK("k_embed_finish");
        });
    });
}

}  // extern "C"
