// Products with 4-bit weights in groups: W[n, k] = s q + b with q in 0..15 and one (s, b) a row and group of 32, 64 or 128
// consecutive k. A sum over a group is s (sum of q x) + b (sum of x), so the integers q go into the matrix instructions as
// they are (exact in 16 bits) and s and b act on fp32 sums once a group: no weight is ever rounded.
//
// Layout (ea_q4_pack): a matrix [N, K] is cut into tiles of 16 rows (the last filled up with zeros) and chunks of 128 k
// (likewise); a tile's chunk is 1024 bytes of words, then 16 rows x 128 / group words (s in the low half, b in the high).
// Lane l of a wave reads the 16 bytes at 16 l of the words: word j holds row l & 15 at k = 32 j + 8 (l >> 4) + 0..7, the B
// operand of the chunk's j-th 16x16x32 product; so a wave's read of a chunk is one contiguous kilobyte. In a word, k + 0..3
// are in the even half-bytes and k + 4..7 in the odd ones: masked by 0x0f0f0f0f, four of them are four bytes q, and a byte
// q < 16 read as e4m3 is q / 512 exactly (below 8 a subnormal), which one conversion with the scale 512 turns into q.
#pragma once

#include <hip/hip_runtime.h>

#include <type_traits>

#include "ea_device.hpp"

namespace ea {

typedef __bf16 b8v __attribute__((ext_vector_type(8)));
typedef u4v u4v_a8 __attribute__((aligned(8)));  // 16 bytes of a row of activations, rows 8-byte aligned

constexpr int Q4_CHUNK = 128, Q4_WORDS = 1024;

// gpc: groups a chunk (4, 2 or 1 for groups of 32, 64, 128)
__host__ __device__ constexpr int q4_chunk_bytes(int gpc) { return Q4_WORDS + 64 * gpc; }
__host__ __device__ inline uint32_t q4_chunks(uint32_t k) { return k / Q4_CHUNK + (k % Q4_CHUNK != 0); }
__host__ __device__ inline uint32_t q4_tiles(uint32_t n) { return n / 16 + (n % 16 != 0); }

template <bool BF>
__device__ __forceinline__ f4v q4_mfma(const u4v& a, const u4v& b, const f4v& c) {
    if constexpr (BF)
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8v, a), __builtin_bit_cast(b8v, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8v, a), __builtin_bit_cast(h8v, b), c, 0, 0, 0);
}

// The eight values of a word as bf16 or fp16 integers.
template <bool BF>
__device__ __forceinline__ u4v q4_values(uint32_t w) {
    const uint32_t lo = w & 0x0f0f0f0fu, hi = (w >> 4) & 0x0f0f0f0fu;
    if constexpr (BF)
        return u4v{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 512.0f, false)),
                   __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 512.0f, true)),
                   __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 512.0f, false)),
                   __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 512.0f, true))};
    else
        return u4v{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 512.0f, false)),
                   __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 512.0f, true)),
                   __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 512.0f, false)),
                   __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 512.0f, true))};
}

template <bool BF>
__device__ __forceinline__ u4v q4_ones() {
    constexpr uint32_t one = BF ? 0x3f803f80u : 0x3c003c00u;
    return u4v{one, one, one, one};
}

// A chunk's (s, b) of the lane's weight row.
template <int GPC>
struct Q4Params {
    uint32_t w[GPC];
};
template <int GPC>
__device__ __forceinline__ Q4Params<GPC> q4_params(const uint8_t* chunk, int lane) {
    return *reinterpret_cast<const Q4Params<GPC>*>(chunk + Q4_WORDS + 4 * GPC * (lane & 15));
}
template <bool SBF>
__device__ __forceinline__ void q4_scale_bias(uint32_t p, float& s, float& b) {
    s = SBF ? __builtin_bit_cast(float, p << 16) : h2f((uint16_t)(p & 0xffffu));
    b = SBF ? __builtin_bit_cast(float, p & 0xffff0000u) : h2f((uint16_t)(p >> 16));
}

// A chunk of NT tiles against 16 rows: out += the chunk's share. a[j]: the rows' A operands of the chunk's four products. The
// sums of x come from the same operands against ones, which leaves them in the accumulators' own layout (lane l: rows
// 4 (l >> 4) + i, weight row l & 15).
template <bool BF, bool SBF, int GPC, int NT>
__device__ __forceinline__ void q4_chunk(const u4v (&words)[NT], const Q4Params<GPC> (&par)[NT], const u4v (&a)[4],
                                         f4v (&out)[NT]) {
    constexpr int JPG = 4 / GPC;
    const f4v zero{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int g = 0; g < GPC; ++g) {
        f4v xs;
#pragma unroll
        for (int j = 0; j < JPG; ++j) xs = q4_mfma<BF>(a[g * JPG + j], q4_ones<BF>(), j ? xs : zero);
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            f4v acc;
#pragma unroll
            for (int j = 0; j < JPG; ++j) acc = q4_mfma<BF>(a[g * JPG + j], q4_values<BF>(words[t][g * JPG + j]), j ? acc : zero);
            float s, b;
            q4_scale_bias<SBF>(par[t].w[g], s, b);
#pragma unroll
            for (int i = 0; i < 4; ++i) out[t][i] = __builtin_fmaf(b, xs[i], __builtin_fmaf(s, acc[i], out[t][i]));
        }
    }
}

// The lane's A operands of one chunk of a row of 16-bit activations (k a multiple of 32). Past k, where the weights, scales
// and biases are zeros, values of the row before it stand in: times zero they add nothing, as long as the row is finite.
__device__ __forceinline__ void q4_rows(const uint16_t* row, uint32_t chunk, uint32_t k, int lane, u4v (&a)[4]) {
    const uint16_t* p = row + (size_t)chunk * Q4_CHUNK + 8 * (lane >> 4);
    const int last = (int)(k - chunk * Q4_CHUNK) - 32;
#pragma unroll
    for (int j = 0; j < 4; ++j) a[j] = (u4v) * reinterpret_cast<const u4v_a8*>(p + min(32 * j, last));
}

// The tiles at w, w + tile_bytes, .. (of a matrix with fewer than NT the last one again) against 16 rows over the chunks c0,
// c0 + step, ..: the loads of NB chunks are issued before the first of their products. With SOME, a lane whose row is null
// reads nothing and multiplies zeros.
template <bool BF, bool SBF, int GPC, int NT, int NB, bool SOME = false>
__device__ __forceinline__ void q4_stream(const uint8_t* w, size_t tile_bytes, uint32_t c0, uint32_t step, uint32_t chunks,
                                          const uint16_t* row, uint32_t k, int lane, f4v (&out)[NT],
                                          uint32_t last_tile = NT - 1) {
    for (uint32_t c = c0; c < chunks; c += step * NB) {
        u4v words[NB][NT], x[NB][4];
        Q4Params<GPC> par[NB][NT];
#pragma unroll
        for (int i = 0; i < NB; ++i) {
            const uint32_t ci = min(c + step * i, chunks - 1);
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                const uint8_t* p = w + min((uint32_t)t, last_tile) * tile_bytes + (size_t)ci * q4_chunk_bytes(GPC);
                words[i][t] = reinterpret_cast<const u4v*>(p)[lane];
                par[i][t] = q4_params<GPC>(p, lane);
            }
            if constexpr (!SOME) q4_rows(row, ci, k, lane, x[i]);
        }
        if constexpr (SOME) {
#pragma unroll
            for (int i = 0; i < NB; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) x[i][j] = u4v{0, 0, 0, 0};
            if (row) {
#pragma unroll
                for (int i = 0; i < NB; ++i) q4_rows(row, min(c + step * i, chunks - 1), k, lane, x[i]);
            }
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < NB; ++i)
            if (c + step * i < chunks) q4_chunk<BF, SBF, GPC, NT>(words[i], par[i], x[i], out);
    }
}

// Value (row r, weight row n of tile t) summed over the waves' parts, in wave order.
template <int WK, int NT>
__device__ __forceinline__ float q4_total(const f4v (&part)[WK][NT][64], int t, int r, int n) {
    const float* all = reinterpret_cast<const float*>(part) + (t * 64 + (r >> 2) * 16 + n) * 4 + (r & 3);
    float v = all[0];
#pragma unroll
    for (int k = 1; k < WK; ++k) v = v + all[k * NT * 256];
    return v;
}

// The sums of NT tiles (lane l: rows 4 (l >> 4) + i, column l & 15 of each) through a wave's own LDS, so that a lane gets four
// neighbouring columns: piece(row, column, four sums) for 16 rows of 16 NT columns, 16 NT / 4 lanes a row. A store then covers
// whole lines, and a wave has a quarter of the stores in flight.
template <int NT>
constexpr int q4_turn_floats() { return 16 * (16 * NT + 4); }
template <int NT, typename F>
__device__ __forceinline__ void q4_turn(float* lds, const f4v (&v)[NT], int lane, F piece) {
    constexpr int STRIDE = 16 * NT + 4, LANES = 4 * NT;
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) lds[(4 * (lane >> 4) + i) * STRIDE + 16 * t + (lane & 15)] = v[t][i];
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // the wave's LDS works in order; the compiler has to as well
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int k = 0; k < NT; ++k) {
        const int at = 64 * k + lane, r = at / LANES, c = 4 * (at % LANES);
        piece(r, c, *reinterpret_cast<const f4v*>(lds + r * STRIDE + c));
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// f(groups a chunk, x in bf16, scales in bf16) as compile-time constants.
template <typename F>
inline void q4_types(bool bf, bool sbf, int gpc, F f) {
    const auto types = [&](auto gpc_) {
        if (bf && sbf) f(gpc_, std::true_type{}, std::true_type{});
        else if (bf) f(gpc_, std::true_type{}, std::false_type{});
        else if (sbf) f(gpc_, std::false_type{}, std::true_type{});
        else f(gpc_, std::false_type{}, std::false_type{});
    };
    if (gpc == 4) types(std::integral_constant<int, 4>{});
    else if (gpc == 2) types(std::integral_constant<int, 2>{});
    else types(std::integral_constant<int, 1>{});
}

}  // namespace ea
