// Sums over the lanes that share a row, and the places in LDS where the waves of a wide row meet.
// Its includer declares row_total (device_common.hpp).
#pragma once

namespace smx {
namespace node {

// The sums of K values over G lanes, in all of them; G a power of two from 16 on, lanes side by
// side, above a wave the whole workgroup, with one barrier a call: a wave past it may be in its next call while another
// still reads, so consecutive calls write the two halves of `room` in turn, and by the call after that every wave has passed
// the barrier of the one between.  That holds for calls with one Room and one `turn`: sums of another K in between have
// both of their own, in other memory.
template <int G, int K>
struct GroupSum {
    static constexpr int kWaves = G > 64 ? G / 64 : 1;
    struct Room {
        float v[2][K][kWaves];
    };
    __device__ __forceinline__ static void sum(float (&v)[K], Room& room, int& turn) {
#pragma unroll
        for (int k = 0; k < K; ++k) {
            v[k] = row_total(v[k]);
            if constexpr (G >= 32) v[k] += __shfl_xor(v[k], 16);
            if constexpr (G >= 64) v[k] += __shfl_xor(v[k], 32);
        }
        if constexpr (G > 64) {
            turn ^= 1;
            if (threadIdx.x % 64 == 0)
#pragma unroll
                for (int k = 0; k < K; ++k) room.v[turn][k][threadIdx.x / 64] = v[k];
            __syncthreads();
            const int w = threadIdx.x % 16;
#pragma unroll
            for (int k = 0; k < K; ++k) v[k] = row_total(w < kWaves ? room.v[turn][k][w] : 0.0f);
        }
    }
};

// The two rounds of sums of a row's gradient, each with a room and a turn of its own.
template <int G>
struct GradientSums {
    struct Room {
        typename GroupSum<G, 1>::Room one;
        typename GroupSum<G, 5>::Room five;
    };
    Room& room;
    int turn_one = 0, turn_five = 0;
    __device__ __forceinline__ void sum(float (&v)[1]) { GroupSum<G, 1>::sum(v, room.one, turn_one); }
    __device__ __forceinline__ void sum(float (&v)[5]) { GroupSum<G, 5>::sum(v, room.five, turn_five); }
};

}  // namespace node
}  // namespace smx
