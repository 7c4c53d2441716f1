// 4-bit products for many rows: a block multiplies 16 MT rows by column blocks of 4 NT tiles, a wave NT tiles by all rows.
// The rows' chunks are staged in LDS for the four waves, in two buffers, while the chunk before is multiplied; a wave's
// weights come straight from memory into registers a chunk ahead. A tile's words are turned into MFMA operands once for
// 16 MT rows, the sums of x once for NT tiles.
#pragma once

#include "ea_q4.hpp"

namespace ea {

constexpr int Q4_GEMM_THREADS = 256;
// LDS: chunks of 16 MT rows with all TERMS of the rows, 4096 MT TERMS bytes each (`resident` of them, or two), their sums over
// eight groups each, 1024 MT bytes (of all groups, or in two buffers), and the waves' places to turn two tiles' sums: behind
// them, or in the place of all.
template <int MT, int TERMS>
constexpr int q4_gemm_lds(int resident = 0, int eights = 2) {
    const int turn = 4 * 4 * q4_turn_floats<2>(), sums = eights * MT * 1024, two = 2 * MT * 4096 * TERMS + sums;
    return resident ? resident * MT * 4096 * TERMS + sums + turn : two > turn ? two : turn;
}
constexpr int Q4_RESIDENT = 65536;  // bytes of chunks that stay in LDS at most, so that a CU holds two blocks

// One chunk from LDS: row r of the block at 256 r, its 16-byte piece q at 16 (q ^ (r & 15)), so that the 16 rows of an
// operand's quarter lie in different banks. With BIAS the groups' biases are applied here, from sums of x that are made here
// too; without, out gets the scaled sums alone. Rows of several TERMS, 4096 MT bytes apart, add up: a weight is turned into an
// operand once for all of them, and their products share an accumulator.
template <bool BF, bool SBF, int GPC, int MT, int NT, bool BIAS, int TERMS = 1>
__device__ __forceinline__ void q4_gemm_chunk(const uint8_t* lds, const u4v (&words)[NT], const Q4Params<GPC> (&par)[NT],
                                              int lane, f4v (&out)[NT][MT]) {
    constexpr int JPG = 4 / GPC;
    const f4v zero{0.0f, 0.0f, 0.0f, 0.0f};
    const int r = lane & 15, quad = lane >> 4;
    if constexpr (TERMS > 1) {
        static_assert(!BIAS, "biases of several terms come from their sums");
#pragma unroll
        for (int g = 0; g < GPC; ++g) {
            f4v acc[NT][MT];
#pragma unroll
            for (int j = 0; j < JPG; ++j) {
                u4v b[NT];
#pragma unroll
                for (int t = 0; t < NT; ++t) b[t] = q4_values<BF>(words[t][g * JPG + j]);
#pragma unroll
                for (int term = 0; term < TERMS; ++term)
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt) {
                        const u4v a = *reinterpret_cast<const u4v*>(lds + ((term * MT + mt) * 16 + r) * 256 +
                                                                    16 * ((4 * (g * JPG + j) + quad) ^ r));
#pragma unroll
                        for (int t = 0; t < NT; ++t) acc[t][mt] = q4_mfma<BF>(a, b[t], j || term ? acc[t][mt] : zero);
                    }
            }
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                float s, b;
                q4_scale_bias<SBF>(par[t].w[g], s, b);
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                    for (int i = 0; i < 4; ++i) out[t][mt][i] = __builtin_fmaf(s, acc[t][mt][i], out[t][mt][i]);
            }
        }
        return;
    }
#pragma unroll
    for (int g = 0; g < GPC; ++g) {
        u4v a[MT][JPG];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int j = 0; j < JPG; ++j)
                a[mt][j] = *reinterpret_cast<const u4v*>(lds + (mt * 16 + r) * 256 + 16 * ((4 * (g * JPG + j) + quad) ^ r));
        f4v xs[MT];
        if constexpr (BIAS) {
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                for (int j = 0; j < JPG; ++j) xs[mt] = q4_mfma<BF>(a[mt][j], q4_ones<BF>(), j ? xs[mt] : zero);
        }
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            f4v acc[MT];
#pragma unroll
            for (int j = 0; j < JPG; ++j) {
                const u4v b = q4_values<BF>(words[t][g * JPG + j]);
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) acc[mt] = q4_mfma<BF>(a[mt][j], b, j ? acc[mt] : zero);
            }
            float s, b;
            q4_scale_bias<SBF>(par[t].w[g], s, b);
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float v = __builtin_fmaf(s, acc[mt][i], out[t][mt][i]);
                    out[t][mt][i] = BIAS ? __builtin_fmaf(b, xs[mt][i], v) : v;
                }
        }
    }
}

// ---- the biases of all groups at once -----------------------------------------------------------------------------------
// Where the rows' sums over each group are known before, biases need no fp32 operations of their own: sums and biases are a
// product over the groups. A sum is held as three bf16 numbers that add up to it (24 bits), for each eight groups 64 bytes: the
// eight first terms, the second, the third, zeros; so a lane's A operand of eight groups is one 16-byte read (lanes 16 q .. are
// term q), the B operand the eight biases, the same for every term, collected from the chunks' parameters as they pass. (Half
// of the loop's fp32 operations went into the biases before, and with four tiles a wave a fifth of its matrix instructions.)
__host__ __device__ inline uint32_t q4_sum_bytes(uint32_t groups) { return (groups + 7) / 8 * 64; }

template <bool SBF, int GPC>
struct Q4Biases {
    u4v hi, lo;  // eight biases in bf16, the last ones at the end; fp16's 11 bits as two of them

    __device__ __forceinline__ void shift(uint32_t h, uint32_t l) {  // two biases, or one in the low half
        if constexpr (GPC == 1) {
            hi = u4v{__builtin_amdgcn_alignbit(hi[1], hi[0], 16), __builtin_amdgcn_alignbit(hi[2], hi[1], 16),
                     __builtin_amdgcn_alignbit(hi[3], hi[2], 16), __builtin_amdgcn_alignbit(h, hi[3], 16)};
            if constexpr (!SBF)
                lo = u4v{__builtin_amdgcn_alignbit(lo[1], lo[0], 16), __builtin_amdgcn_alignbit(lo[2], lo[1], 16),
                         __builtin_amdgcn_alignbit(lo[3], lo[2], 16), __builtin_amdgcn_alignbit(l, lo[3], 16)};
        } else {
            hi = u4v{hi[1], hi[2], hi[3], h};
            if constexpr (!SBF) lo = u4v{lo[1], lo[2], lo[3], l};
        }
    }
    // A chunk's biases.
    __device__ __forceinline__ void take(const Q4Params<GPC>& par) {
#pragma unroll
        for (int g = 0; g < GPC; g += 2) {
            const uint32_t w0 = par.w[g], w1 = GPC == 1 ? 0u : par.w[g + (GPC > 1)];
            if constexpr (SBF) {
                shift((w0 >> 16) | (w1 & 0xffff0000u), 0);
            } else {
                // fp16's 11 bits: the upper 8 as they stand, which leaves 3
                const float a = h2f((uint16_t)(w0 >> 16)), b = h2f((uint16_t)(w1 >> 16));
                const uint32_t ah = __builtin_bit_cast(uint32_t, a) & 0xffff0000u, bh = __builtin_bit_cast(uint32_t, b) & 0xffff0000u;
                const uint32_t al = __builtin_bit_cast(uint32_t, a - __builtin_bit_cast(float, ah));
                const uint32_t bl = __builtin_bit_cast(uint32_t, b - __builtin_bit_cast(float, bh));
                shift(ah >> 16 | bh, al >> 16 | (bl & 0xffff0000u));
            }
        }
    }
    template <int MT>
    __device__ __forceinline__ void add(const u4v (&sums)[MT], f4v (&out)[MT]) const {
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
            out[mt] = q4_mfma<true>(sums[mt], hi, out[mt]);
            if constexpr (!SBF) out[mt] = q4_mfma<true>(sums[mt], lo, out[mt]);
        }
    }
};

// A row's sums over its groups, in that form, by `parts` waves of which this is one, eight values a lane; `terms` of the row,
// `plane` values apart.
template <bool BF>
__device__ __forceinline__ void q4_row_sums(const uint16_t* row, uint32_t terms, size_t plane, uint32_t k, uint32_t group,
                                            uint8_t* to, int lane, uint32_t part, uint32_t parts) {
    const uint32_t groups = k / group, per = group / 8, padded = (groups + 7) / 8 * 8;
    for (uint32_t p = 64 * part + lane; p - lane < padded * per; p += 64 * parts) {  // a piece of eight values
        float v = 0.0f;
        if (p < k / 8)
            for (uint32_t t = 0; t < terms; ++t) {
                const u4v u = *reinterpret_cast<const u4v_a8*>(row + t * plane + 8 * p);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    v = v + (BF ? bf2f((uint16_t)(u[i] & 0xffffu)) : h2f((uint16_t)(u[i] & 0xffffu)));
                    v = v + (BF ? bf2f((uint16_t)(u[i] >> 16)) : h2f((uint16_t)(u[i] >> 16)));
                }
            }
        v = v + lane_xor<1>(v);
        v = v + lane_xor<2>(v);
        if (per >= 8) v = v + lane_xor<4>(v);
        if (per >= 16) v = v + lane_xor<8>(v);
        const uint32_t g = p / per;
        if (p % per == 0 && g < padded) {
            uint16_t* o = reinterpret_cast<uint16_t*>(to + (size_t)(g / 8) * 64) + (g & 7);
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                const uint16_t b = t < 3 ? f2bf(v) : 0;
                o[8 * t] = b;
                v = __builtin_fabsf(v) < __builtin_inff() ? v - bf2f(b) : 0.0f;
            }
        }
    }
}

// The column blocks cb, cb + cb_step, .. of W (its first tile at w) times the block's rows. row(i): row i's activations,
// TERMS of them `plane` values apart (their products add up); sums(i): its groups' sums, for the biases. With TURN store(row,
// column of W's packed rows, the sums of four columns), else store(tile, the lane's sums). RESIDENT: all of the rows' terms and
// chunks lie in LDS at once (Q4_RESIDENT bytes at most), so that after the first barrier the waves go on alone; else two
// chunks do. Weights are read a chunk before their products.
template <bool BF, bool SBF, int GPC, int MT, int NT, int TERMS, bool RESIDENT, bool TURN, typename ROW, typename SUMS,
          typename STORE>
__device__ __forceinline__ void q4_gemm(uint8_t* lds, const uint8_t* w, uint32_t tiles, uint32_t k, size_t plane,
                                        uint32_t cb, uint32_t cb_step, ROW row, SUMS sums, STORE store) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t chunks = q4_chunks(k), piece = threadIdx.x & 15, row0 = threadIdx.x >> 4;
    const uint32_t tile_bytes = chunks * q4_chunk_bytes(GPC);
    constexpr uint32_t CYCLE = 8 / GPC;  // chunks of eight groups
    constexpr uint32_t BUFFER = TERMS * MT * 4096;
    const uint16_t* src[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) src[i] = row(row0 + 16 * i);
    // the sums' 16-byte pieces, one a thread: row threadIdx / 4, piece threadIdx % 4 at 16 (4 row + (piece ^ (row / 4 & 3)))
    const uint32_t srow = threadIdx.x >> 2, sto = 16 * (4 * srow + ((threadIdx.x & 3) ^ (srow >> 2 & 3)));
    const uint8_t* const rs = sums(min(srow, 16u * MT - 1)) + 16 * (threadIdx.x & 3);
    uint8_t* const lds_sums = lds + (RESIDENT ? chunks : 2) * BUFFER;
    const uint32_t to = row0 * 256 + 16 * (piece ^ row0);  // row0 + 16 i: 4096 bytes further each
    u4v ra[TERMS][MT], rw[2][NT], rx{};
    Q4Params<GPC> rp[2][NT];
    Q4Biases<SBF, GPC> biases[NT];
    struct Cursor {
        uint32_t cb, c;
    };
    const auto next = [&](Cursor at) {
        if (++at.c == chunks) at.c = 0, at.cb += cb_step;
        return at;
    };
    const auto inside = [&](const Cursor& at) { return at.cb * 4 * NT < tiles; };
    const auto load_rows = [&](uint32_t c) {
        // past k, where the weights are zeros, the row's last 32 values again
        const uint32_t at = c * Q4_CHUNK + 8 * piece, off = at < k ? at : k - 32 + 8 * (piece & 3);
#pragma unroll
        for (int t = 0; t < TERMS; ++t)
#pragma unroll
            for (int i = 0; i < MT; ++i) ra[t][i] = *reinterpret_cast<const u4v_a8*>(src[i] + t * plane + off);
    };
    const auto stage = [&](uint32_t buffer) {
#pragma unroll
        for (int t = 0; t < TERMS; ++t)
#pragma unroll
            for (int i = 0; i < MT; ++i) *reinterpret_cast<u4v*>(lds + buffer * BUFFER + to + 4096 * (t * MT + i)) = ra[t][i];
    };
    const auto load = [&](int set, const Cursor& at) {
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const uint32_t tile = min((at.cb * 4 + wave) * NT + t, tiles - 1);
            const uint8_t* p = w + (size_t)tile * tile_bytes + (size_t)at.c * q4_chunk_bytes(GPC);
            rw[set][t] = reinterpret_cast<const u4v*>(p)[lane];
            rp[set][t] = q4_params<GPC>(p, lane);
        }
    };
    f4v out[NT][MT];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) out[t][mt] = f4v{0.0f, 0.0f, 0.0f, 0.0f};
    Cursor at{cb, 0};
    uint32_t buffer = 0;
    // one chunk; false after the last
    const auto step = [&](auto set_) __attribute__((always_inline)) {
        constexpr int SET = decltype(set_)::value;
        const uint32_t c = at.c;
        if constexpr (!RESIDENT) stage(buffer);
        const bool ends = c + 1 == chunks;  // of the column block
        const Cursor then = next(at);
        const bool more = inside(then);
        // Eight groups' sums are read with the first of their chunks, and go to LDS a chunk later (a barrier after the other
        // buffer's last readers), or at once if no chunk follows: with one chunk in all, over the same values.
        uint8_t* const cycle_sums = lds_sums + (RESIDENT ? c / CYCLE : c / CYCLE & 1) * (MT * 1024);
        if constexpr (!RESIDENT) {
            if (c % CYCLE == 0) rx = *reinterpret_cast<const u4v*>(rs + c / CYCLE * 64);
            if ((c % CYCLE == 1 || (c % CYCLE == 0 && ends)) && srow < 16u * MT)
                *reinterpret_cast<u4v*>(cycle_sums + sto) = rx;
            if (more) load_rows(then.c);
        }
        if (more) load(1 - SET, then);
        if constexpr (!RESIDENT) __syncthreads();  // the chunk is staged; its buffer's last readers were before the last one
        q4_gemm_chunk<BF, SBF, GPC, MT, NT, false, TERMS>(lds + (RESIDENT ? c : buffer) * BUFFER, rw[SET], rp[SET], lane, out);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int t = 0; t < NT; ++t) biases[t].take(rp[SET][t]);
        if (c % CYCLE == CYCLE - 1 || ends) {
            for (uint32_t i = c % CYCLE; i < CYCLE - 1; ++i) {  // no more chunks: zeros up to the eighth group
                constexpr Q4Params<GPC> none{};
#pragma unroll
                for (int t = 0; t < NT; ++t) biases[t].take(none);
            }
            u4v a[MT];
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
                const int r = mt * 16 + (lane & 15);
                a[mt] = *reinterpret_cast<const u4v*>(cycle_sums + 16 * (4 * r + ((lane >> 4) ^ (r >> 2 & 3))));
            }
#pragma unroll
            for (int t = 0; t < NT; ++t) biases[t].add(a, out[t]);
        }
        if (ends) {
            const uint32_t tile0 = (at.cb * 4 + wave) * NT;
            if constexpr (TURN) {  // 16 rows of the wave's columns at a time, where the chunks were once no wave reads them
                if constexpr (!RESIDENT) __syncthreads();
                static_assert(NT % 2 == 0);
                float* const mine = reinterpret_cast<float*>(RESIDENT ? lds_sums + (chunks + CYCLE - 1) / CYCLE * (MT * 1024) : lds) +
                                    wave * q4_turn_floats<2>();
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                    for (int t = 0; t < NT; t += 2) {
                        const f4v v[2] = {out[t][mt], out[t + 1][mt]};
                        q4_turn<2>(mine, v, lane, [&](int r, int c, const f4v& p) {
                            if (tile0 + t + c / 16 < tiles) store(16 * mt + r, (tile0 + t) * 16 + c, p);
                        });
                    }
                if constexpr (!RESIDENT)
                    if (more) __syncthreads();
            } else {
#pragma unroll
                for (int t = 0; t < NT; ++t)
                    if (tile0 + t < tiles) store(tile0 + t, out[t]);
            }
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) out[t][mt] = f4v{0.0f, 0.0f, 0.0f, 0.0f};
        }
        at = then;
        buffer ^= 1;
        return more;
    };
    if constexpr (!RESIDENT) load_rows(0);
    load(0, at);
    if constexpr (RESIDENT) {
        for (uint32_t ci = 0; ci < chunks; ++ci) {
            load_rows(ci);
            stage(ci);
        }
        for (uint32_t i = 0; i * CYCLE < chunks; ++i)
            if (srow < 16u * MT)
                *reinterpret_cast<u4v*>(lds_sums + i * (MT * 1024) + sto) = *reinterpret_cast<const u4v*>(rs + i * 64);
        __syncthreads();
    }
    while (step(std::integral_constant<int, 0>{}) && step(std::integral_constant<int, 1>{})) {
    }
}

}  // namespace ea
