// 4-bit products for many rows: a block multiplies 16 MT rows by column blocks of 4 NT tiles, a wave NT tiles by all rows.
// The rows' chunks are staged in LDS for the four waves, in two buffers, while the chunk before is multiplied; a wave's
// weights come straight from memory into registers a chunk ahead. A tile's words are turned into MFMA operands once for
// 16 MT rows, the sums of x once for NT tiles.
#pragma once

#include "ea_q4.hpp"

namespace ea {

constexpr int Q4_GEMM_THREADS = 256;
template <int MT>
constexpr int q4_gemm_lds() { return 2 * MT * 16 * 256; }

// One chunk from LDS: row r of the block at 256 r, its 16-byte piece q at 16 (q ^ (r & 15)), so that the 16 rows of an
// operand's quarter lie in different banks.
template <bool BF, bool SBF, int GPC, int MT, int NT>
__device__ __forceinline__ void q4_gemm_chunk(const uint8_t* lds, const u4v (&words)[NT], const Q4Params<GPC> (&par)[NT],
                                              int lane, f4v (&out)[NT][MT]) {
    constexpr int JPG = 4 / GPC;
    const f4v zero{0.0f, 0.0f, 0.0f, 0.0f};
    const int r = lane & 15, quad = lane >> 4;
#pragma unroll
    for (int g = 0; g < GPC; ++g) {
        u4v a[MT][JPG];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int j = 0; j < JPG; ++j)
                a[mt][j] = *reinterpret_cast<const u4v*>(lds + (mt * 16 + r) * 256 + 16 * ((4 * (g * JPG + j) + quad) ^ r));
        f4v xs[MT];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int j = 0; j < JPG; ++j) xs[mt] = q4_mfma<BF>(a[mt][j], q4_ones<BF>(), j ? xs[mt] : zero);
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
                for (int i = 0; i < 4; ++i)
                    out[t][mt][i] = __builtin_fmaf(b, xs[mt][i], __builtin_fmaf(s, acc[mt][i], out[t][mt][i]));
        }
    }
}

// The column blocks cb, cb + cb_step, .. of W (its first tile at w) times the block's rows. row(i): row i's activations,
// terms of them `plane` values apart (their products add up). store(tile, sums of its 16 MT rows).
template <bool BF, bool SBF, int GPC, int MT, int NT, typename ROW, typename STORE>
__device__ __forceinline__ void q4_gemm(uint8_t* lds, const uint8_t* w, uint32_t tiles, uint32_t k, uint32_t terms,
                                        size_t plane, uint32_t cb, uint32_t cb_step, ROW row, STORE store) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t chunks = q4_chunks(k), piece = threadIdx.x & 15, row0 = threadIdx.x >> 4;
    const size_t tile_bytes = (size_t)chunks * q4_chunk_bytes(GPC);
    const uint16_t* src[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) src[i] = row(row0 + 16 * i);
    const uint32_t to = row0 * 256 + 16 * (piece ^ row0);  // row0 + 16 i: 4096 bytes further each
    u4v ra[MT], rw[NT];
    Q4Params<GPC> rp[NT];
    const auto load = [&](uint32_t cb_, uint32_t term, uint32_t c) {
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const uint32_t tile = min((cb_ * 4 + wave) * NT + t, tiles - 1);
            const uint8_t* p = w + tile * tile_bytes + (size_t)c * q4_chunk_bytes(GPC);
            rw[t] = reinterpret_cast<const u4v*>(p)[lane];
            rp[t] = q4_params<GPC>(p, lane);
        }
        // past k, where the weights are zeros, the row's last 32 values again
        const uint32_t at = c * Q4_CHUNK + 8 * piece, off = at < k ? at : k - 32 + 8 * (piece & 3);
#pragma unroll
        for (int i = 0; i < MT; ++i) ra[i] = *reinterpret_cast<const u4v_a8*>(src[i] + term * plane + off);
    };
    const auto stage = [&](uint32_t buffer) {
#pragma unroll
        for (int i = 0; i < MT; ++i) *reinterpret_cast<u4v*>(lds + buffer * (MT * 4096) + to + 4096 * i) = ra[i];
    };
    f4v out[NT][MT];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) out[t][mt] = f4v{0.0f, 0.0f, 0.0f, 0.0f};
    uint32_t c = 0, term = 0, buffer = 0;
    load(cb, 0, 0);
    stage(0);
    for (;;) {
        const bool ends = c + 1 == chunks && term + 1 == terms;  // of the column block
        uint32_t nc = c + 1, nterm = term, ncb = cb;
        if (nc == chunks) nc = 0, ++nterm;
        if (nterm == terms) nterm = 0, ncb += cb_step;
        const bool more = ncb * 4 * NT < tiles;
        u4v words[NT];
        Q4Params<GPC> par[NT];
#pragma unroll
        for (int t = 0; t < NT; ++t) words[t] = rw[t], par[t] = rp[t];
        if (more) load(ncb, nterm, nc);
        __syncthreads();  // the chunk is staged, and the buffer of the one before it is free
        q4_gemm_chunk<BF, SBF, GPC, MT, NT>(lds + buffer * (MT * 4096), words, par, lane, out);
        if (ends) {
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                const uint32_t tile = (cb * 4 + wave) * NT + t;
                if (tile < tiles) store(tile, out[t]);
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) out[t][mt] = f4v{0.0f, 0.0f, 0.0f, 0.0f};
            }
        }
        if (!more) break;
        buffer ^= 1;
        stage(buffer);
        c = nc;
        term = nterm;
        cb = ncb;
    }
}

}  // namespace ea
