// Routed experts with 4-bit weights in groups: out[r] = sum over slots of wts * down_e(silu(gate_e x) * (up_e x)).
//
// The rows' picks are sorted by expert and cut into items (an expert and up to 16 of its pairs); a block multiplies an
// item's rows by tiles of the expert's gate|up (8 columns of each) and writes the activated pairs; another multiplies those
// by tiles of the down projection; the last launch adds a row's slots in order. A pair's values depend neither on the others
// of its item nor on their order, so the results are the same on every run. Where experts have many rows, items are of up
// to 64 pairs (long items), which turn a weight into a matrix operand once for all of them.
//
// A pair takes 6 D I operations, an expert that is picked 3 D I / 2 bytes of words and 12 D I / group of scales and biases: up
// to some tens of rows the weights' bytes bound it, at one row latencies. Figures in this file: D 6144, I 256, 256 experts,
// 8 picks a row (even ones up to 512 rows, Zipf 1.1 above), groups of 64, bf16 in and out: 1.77 MB gate|up and 0.88 MB down an
// expert.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "ea_host.hpp"
#include "ea_q4_gemm.hpp"

namespace ea {

// dims and width are multiples of a group, so of 32 (q4_experts_ok): gate|up has width / 8 tiles, four or more, down dims / 16,
// two or more, none of them with rows behind its matrix.
constexpr uint32_t Q4_MAX_EXPERTS = 4096;
constexpr uint32_t Q4_ITEM = 16, Q4_BIG_ITEM = 64;         // pairs an item
constexpr uint32_t Q4_ROWS = 16, Q4_PAIRS = Q4_ROWS * 32;  // rows and pairs that are grouped beside the first products

// An expert and up to Q4_ITEM or Q4_BIG_ITEM of its pairs (row * slots + slot).
struct Q4Item {
    int32_t expert, count;
    int32_t pair[Q4_BIG_ITEM];
};

struct Q4MoeArgs {
    const uint16_t* x;
    size_t x_stride;
    const int32_t* pick;
    const float* wts;
    const uint8_t *gu, *down;
    size_t gu_bytes, down_bytes;  // one expert's
    int32_t* nitems;              // items, full ones among them
    Q4Item* items;
    uint16_t* h;                  // bf16 [terms][pairs][width], terms 2 or 3
    uint8_t *xsums, *hsums;       // sums over groups of a row of x, of a pair of h (q4_row_sums)
    float* y;                     // fp32 [pairs][dims]
    void* out;
    uint32_t rows, pairs, dims, width, experts, slots, item;  // item: pairs an item at most
    int out_dtype, terms;
    uint32_t group;
    bool bf;
};

// ---- grouping -----------------------------------------------------------------------------------------------------
// One block: the pairs of each expert counted, the items before each expert scanned, the pairs placed (in any order within an
// expert). Full items come before all others, so that the longest work starts first. A pick outside 0 .. experts - 1 is a slot
// without an expert. Bound by its passes' latencies: 5 us at 64 rows, 8 at 512, 15 at 2048 (with items in four classes of
// size instead of two 24, and 3 % less in the products behind).
__device__ void q4_group(const Q4MoeArgs& a) {
    __shared__ uint32_t count[Q4_MAX_EXPERTS], full[Q4_MAX_EXPERTS], rest[Q4_MAX_EXPERTS], sums[2][16], all;
    __shared__ uint16_t nfull[Q4_MAX_EXPERTS];  // at most EA_Q4_MAX_PAIRS / Q4_ITEM
    constexpr int KEEP = 16;  // picks a thread keeps between the passes
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    uint32_t kept[KEEP];
#pragma unroll
    for (int i = 0; i < KEEP; ++i) kept[i] = (uint32_t)(t + 1024u * i) < a.pairs ? (uint32_t)a.pick[t + 1024 * i] : 0xffffffffu;
    for (uint32_t e = t; e < a.experts; e += 1024) count[e] = 0;
    if (t == 0) all = 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < KEEP; ++i)
        if (kept[i] < a.experts) atomicAdd(&count[kept[i]], 1u);
    for (uint32_t p = t + 1024 * KEEP; p < a.pairs; p += 1024) {
        const uint32_t e = (uint32_t)a.pick[p];
        if (e < a.experts) atomicAdd(&count[e], 1u);
    }
    __syncthreads();
    uint32_t mine = 0;
    for (uint32_t e = t; e < a.experts; e += 1024) mine += count[e] / a.item;
    if (mine) atomicAdd(&all, mine);
    __syncthreads();
    uint32_t fbase = 0, rbase = all;
    for (uint32_t e0 = 0; e0 < a.experts; e0 += 1024) {  // exclusive scans, 1024 experts a step
        const uint32_t e = e0 + t, c = e < a.experts ? count[e] : 0, n = c / a.item, r = c % a.item != 0;
        uint32_t v = n, w = r;
        for (int d = 1; d < 64; d <<= 1) {
            const uint32_t ov = __shfl_up(v, d), ow = __shfl_up(w, d);
            v += lane >= d ? ov : 0;
            w += lane >= d ? ow : 0;
        }
        if (lane == 63) sums[0][wave] = v, sums[1][wave] = w;
        __syncthreads();
        uint32_t fi = fbase + v - n, ri = rbase + w - r;
        for (int i = 0; i < 16; ++i) {
            fi += i < wave ? sums[0][i] : 0;
            ri += i < wave ? sums[1][i] : 0;
            fbase += sums[0][i];
            rbase += sums[1][i];
        }
        if (e < a.experts) {
            full[e] = fi;
            rest[e] = ri;
            nfull[e] = (uint16_t)n;
            count[e] = 0;
        }
        for (uint32_t i = 0; i < n; ++i) {
            a.items[fi + i].expert = (int32_t)e;
            a.items[fi + i].count = (int32_t)a.item;
        }
        if (r) {
            a.items[ri].expert = (int32_t)e;
            a.items[ri].count = (int32_t)(c % a.item);
        }
        __syncthreads();
    }
    const uint32_t base = rbase;
    if (t == 0) a.nitems[0] = (int32_t)base, a.nitems[1] = (int32_t)all;
    const auto place = [&](uint32_t p, uint32_t e) {
        const uint32_t at = atomicAdd(&count[e], 1u), i = at / a.item;
        a.items[i < nfull[e] ? full[e] + i : rest[e]].pair[at % a.item] = (int32_t)p;
    };
#pragma unroll
    for (int i = 0; i < KEEP; ++i)
        if (kept[i] < a.experts) place(t + 1024 * i, kept[i]);
    for (uint32_t p = t + 1024 * KEEP; p < a.pairs; p += 1024) {
        const uint32_t e = (uint32_t)a.pick[p];
        if (e < a.experts) place(p, e);
    }
}

// The grouping, and with more blocks beside it the rows' sums over groups, four waves a row: with one, whose loads come one
// after another, both take 12.5 us at 512 rows in place of 8.0.
constexpr uint32_t Q4_SUM_WAVES = 4;
__global__ void __launch_bounds__(1024) q4_group_kernel(Q4MoeArgs a) {
    if (blockIdx.x == 0) {
        q4_group(a);
        return;
    }
    const uint32_t w = (blockIdx.x - 1) * 16 + (threadIdx.x >> 6), i = w / Q4_SUM_WAVES, part = w % Q4_SUM_WAVES;
    if (i >= a.rows) return;
    uint8_t* to = a.xsums + (size_t)i * q4_sum_bytes(a.dims / a.group);
    const uint16_t* row = a.x + (size_t)i * a.x_stride;
    if (a.bf) q4_row_sums<true>(row, 1, 0, a.dims, a.group, to, threadIdx.x & 63, part, Q4_SUM_WAVES);
    else q4_row_sums<false>(row, 1, 0, a.dims, a.group, to, threadIdx.x & 63, part, Q4_SUM_WAVES);
}

// The same for up to 16 rows, in the order of the experts' first pairs, by a block beside the first products (picks: the
// call's, in LDS, changed). An expert is one item, and a row that names it again is left out: the last launch gives its
// weight to the first naming.
template <int THREADS>
__device__ void q4_group_rows(const Q4MoeArgs& a, int32_t* picks) {
    __shared__ int16_t owner[Q4_PAIRS], before[Q4_PAIRS], index[Q4_PAIRS];
    int32_t once[(Q4_PAIRS + THREADS - 1) / THREADS];
    for (uint32_t p = threadIdx.x, i = 0; p < a.pairs; p += THREADS, ++i) {
        int32_t e = picks[p];
        e = (uint32_t)e < a.experts ? e : -1;
        for (uint32_t q = p - p % a.slots; q < p; ++q) e = picks[q] == e ? -1 : e;
        once[i] = e;
    }
    __syncthreads();
    for (uint32_t p = threadIdx.x, i = 0; p < a.pairs; p += THREADS, ++i) picks[p] = once[i];
    __syncthreads();
    for (uint32_t p = threadIdx.x; p < a.pairs; p += THREADS) {
        const int32_t e = picks[p];
        uint32_t n = 0, own = p;
        if (e >= 0) {
#pragma unroll 4
            for (uint32_t q = 0; q < p; ++q) {
                const bool same = picks[q] == e;
                own = same && n == 0 ? q : own;
                n += same;
            }
        }
        owner[p] = (int16_t)own;
        before[p] = e >= 0 ? (int16_t)n : -1;
    }
    __syncthreads();
    if (threadIdx.x < 64) {
        int items = 0;
        for (uint32_t p0 = 0; p0 < a.pairs; p0 += 64) {
            const uint32_t p = p0 + threadIdx.x;
            const bool fresh = p < a.pairs && before[p] == 0;
            const uint64_t all = __ballot(fresh);
            if (fresh) {
                index[p] = (int16_t)(items + __builtin_popcountll(all & ((1ull << threadIdx.x) - 1)));
                a.items[index[p]].expert = picks[p];
                a.items[index[p]].count = 0;
            }
            items += __builtin_popcountll(all);
        }
        if (threadIdx.x == 0) *a.nitems = items;
    }
    __syncthreads();
    for (uint32_t p = threadIdx.x; p < a.pairs; p += THREADS)
        if (before[p] >= 0) {
            Q4Item& it = a.items[index[owner[p]]];
            it.pair[before[p]] = (int32_t)p;
            atomicMax(&it.count, before[p] + 1);
        }
}

__device__ __forceinline__ float swiglu(float g, float u) { return g / (1.0f + expf_path(0.0f - g)) * u; }

// An activated value as bf16 numbers that add up to it (8 bits each).
__device__ __forceinline__ void store_terms(uint16_t* h, int terms, size_t plane, size_t at, float v) {
    for (int i = 0; i < terms; ++i) {
        const uint16_t b = f2bf(v);
        h[(size_t)i * plane + at] = b;
        v = __builtin_fabsf(v) < __builtin_inff() ? v - bf2f(b) : 0.0f;
    }
}

// ---- gate | up ------------------------------------------------------------------------------------------------------
// Block (NT tiles of gate | up, item): 16 rows of a matrix instruction, those that the item does not have as zeros, which
// cost neither loads nor cache; WK waves take every WK-th chunk. Up to 16 rows nothing is sorted before: block (tiles, pair)
// works if no earlier pair names its expert, a row of the instruction is the row of x, and one more block groups the pairs
// for the launches behind. One row: 6.0 us (2.4 TB/s; the launch, the pick, the weights, the sums after each other). 16 rows
// 43 us (102 experts, 4.2 TB/s), 64 rows, in items, 77 us (5.1 TB/s, above what a large copy reaches). From two rows on two
// tiles a block share their reads of x: 2 / 4 / 8 / 16 rows 9.7 / 14.1 / 25.8 / 42.7 us, with one tile 10.4 / 16.6 / 31.7 /
// 55.6.
enum Q4Rows { ONE_ROW, FEW_ROWS, ITEMS };

template <bool BF, bool SBF, int GPC, int NT, int WK, int NB, int MODE>
__global__ void __launch_bounds__(64 * WK) q4_gateup_kernel(Q4MoeArgs a) {
    __shared__ f4v part[WK][NT][64];
    __shared__ int32_t picks[MODE == FEW_ROWS ? Q4_PAIRS : 16];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t u = blockIdx.y, chunks = q4_chunks(a.dims), r = lane & 15;
    int32_t e;
    const uint16_t* row = nullptr;
    int count = 0;
    if constexpr (MODE == ONE_ROW) {  // every slot by itself: nothing is compared before the weights are read
        e = a.pick[u];
        if ((uint32_t)e >= a.experts) return;
        if (r == 0) row = a.x;
    } else if constexpr (MODE == FEW_ROWS) {
        for (uint32_t p = threadIdx.x; p < a.pairs; p += 64 * WK) picks[p] = a.pick[p];
        __syncthreads();
        if (u == a.pairs) {
            if (blockIdx.x == 0) q4_group_rows<64 * WK>(a, picks);
            return;
        }
        e = picks[u];
        if ((uint32_t)e >= a.experts) return;
        bool before = false;
        for (uint32_t p = lane; p < u; p += 64) before |= picks[p] == e;
        if (__ballot(before)) return;
        if (r < a.rows)
            for (uint32_t k = 0; k < a.slots; ++k)
                if (picks[r * a.slots + k] == e) row = a.x + (size_t)r * a.x_stride;
    } else {
        const Q4Item& it = a.items[u];
        const int n = *a.nitems, p = it.pair[r];  // read together; what lies behind the items is not used
        e = it.expert;
        count = it.count;
        if ((int)u >= n) return;
        if (threadIdx.x < 16) picks[r] = p;
        if ((int)r < count) row = a.x + (size_t)((uint32_t)p / a.slots) * a.x_stride;
    }
    const uint32_t tile0 = blockIdx.x * NT;
    const size_t tile_bytes = (size_t)chunks * q4_chunk_bytes(GPC);
    f4v out[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) out[t] = f4v{0.0f, 0.0f, 0.0f, 0.0f};
    q4_stream<BF, SBF, GPC, NT, NB, true>(a.gu + (size_t)e * a.gu_bytes + tile0 * tile_bytes, tile_bytes, wave, WK, chunks, row,
                                        a.dims, lane, out);
#pragma unroll
    for (int t = 0; t < NT; ++t) part[wave][t][lane] = out[t];
    __syncthreads();
    for (int i = threadIdx.x; i < 128 * NT; i += 64 * WK) {
        const int n = i & 7, t = (i >> 3) % NT, m = i / (8 * NT);
        const uint32_t col = (tile0 + t) * 8 + n;
        uint32_t p = u;
        bool is = true;
        if constexpr (MODE == ONE_ROW) is = m == 0;
        if constexpr (MODE == FEW_ROWS) {  // the row's first naming of the expert
            p = m * a.slots;
            const uint32_t end = (uint32_t)m < a.rows ? p + a.slots : p;
            while (p < end && picks[p] != e) ++p;
            is = p < end;
        }
        if constexpr (MODE == ITEMS) {
            p = picks[m];
            is = m < count;
        }
        if (!is) continue;
        const float v = swiglu(q4_total<WK, NT>(part, t, m, n), q4_total<WK, NT>(part, t, m, n + 8));
        store_terms(a.h, a.terms, (size_t)a.pairs * a.width, (size_t)p * a.width + col, v);
    }
}

// ---- down -----------------------------------------------------------------------------------------------------------
// One row: NT tiles of the output a block; its waves take the (slot, chunk) units in turn, weigh their sums in registers, and
// terms (rows 0 .. TERMS - 1 of the instruction) and waves are added at the end: nothing is left for a launch behind.
// 4.9 us (1.4 TB/s): the launch, picks, weights and sums after each other.
template <bool SBF, int GPC, int TERMS, int NT, int WK, int NB>
__global__ void __launch_bounds__(64 * WK) q4_down_one_kernel(Q4MoeArgs a) {
    __shared__ f4v part[WK][NT][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), term = lane & 15;
    const uint32_t chunks = q4_chunks(a.width), units = a.slots * chunks;
    const uint32_t tile0 = blockIdx.x * NT;
    const size_t tile_bytes = (size_t)chunks * q4_chunk_bytes(GPC), plane = (size_t)a.slots * a.width;
    f4v out[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) out[t] = f4v{0.0f, 0.0f, 0.0f, 0.0f};
    for (uint32_t u0 = wave; u0 < units; u0 += WK * NB) {
        u4v words[NB][NT], x[NB][4];
        Q4Params<GPC> par[NB][NT];
        int32_t e[NB];
        float w[NB];
#pragma unroll
        for (int i = 0; i < NB; ++i) {
            const uint32_t slot = min(u0 + WK * i, units - 1) / chunks;
            e[i] = a.pick[slot];
            w[i] = a.wts[slot];
        }
#pragma unroll
        for (int i = 0; i < NB; ++i) {
            const uint32_t u = min(u0 + WK * i, units - 1), c = u % chunks;
            const uint8_t* p = a.down + (size_t)((uint32_t)e[i] < a.experts ? e[i] : 0) * a.down_bytes + tile0 * tile_bytes +
                               (size_t)c * q4_chunk_bytes(GPC);
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                words[i][t] = reinterpret_cast<const u4v*>(p + t * tile_bytes)[lane];
                par[i][t] = q4_params<GPC>(p + t * tile_bytes, lane);
            }
        }
#pragma unroll
        for (int i = 0; i < NB; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) x[i][j] = u4v{0, 0, 0, 0};
        if (term < TERMS) {
#pragma unroll
            for (int i = 0; i < NB; ++i) {
                const uint32_t u = min(u0 + WK * i, units - 1);
                q4_rows(a.h + term * plane + (size_t)(u / chunks) * a.width, u % chunks, a.width, lane, x[i]);
            }
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < NB; ++i) {
            if (u0 + WK * i >= units || (uint32_t)e[i] >= a.experts) continue;
            f4v y[NT];
#pragma unroll
            for (int t = 0; t < NT; ++t) y[t] = f4v{0.0f, 0.0f, 0.0f, 0.0f};
            q4_chunk<true, SBF, GPC, NT>(words[i], par[i], x[i], y);
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int r = 0; r < TERMS; ++r) out[t][r] = __builtin_fmaf(w[i], y[t][r], out[t][r]);
        }
    }
#pragma unroll
    for (int t = 0; t < NT; ++t) part[wave][t][lane] = out[t];
    __syncthreads();
    for (int i = threadIdx.x; i < 16 * NT; i += 64 * WK) {
        const int n = i & 15, t = i >> 4;
        float v = q4_total<WK, NT>(part, t, TERMS - 1, n);
#pragma unroll
        for (int r = TERMS - 2; r >= 0; --r) v = v + q4_total<WK, NT>(part, t, r, n);  // the small terms first
        store_act(a.out, a.out_dtype, (tile0 + t) * 16 + n, v);
    }
}

// More rows: block (WK NT tiles, item), a wave its NT tiles over all of the width, so that no sum crosses waves and an
// expert's weights are read where they lie together (blocks that took some tiles of every expert read them at half the rate).
// Terms are rows of their own: rows 4 q .. 4 q + 3 of the instruction are quad q of the accumulators' lanes; with three
// terms quad q holds term q of four pairs, with two quads 2 q and 2 q + 1 term q of eight, and adding lanes 16 (and 32)
// apart adds the terms. 16 rows 24 us (3.8 TB/s), 64 rows 46 us (4.3 TB/s): the weights, and a pair's fp32 sums, 24 KB each.
template <bool SBF, int GPC, int TERMS, int NT, int WK, int NB>
__global__ void __launch_bounds__(64 * WK) q4_down_kernel(Q4MoeArgs a) {
    constexpr int PER = TERMS == 2 ? 8 : 4;  // pairs a product
    __shared__ float turn[WK][q4_turn_floats<NT>()];
    const Q4Item& it = a.items[blockIdx.y];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n = *a.nitems, e = it.expert, count = it.count;
    const int from = it.pair[lane & (PER - 1)];
    if ((int)blockIdx.y >= n) return;
    const uint32_t chunks = q4_chunks(a.width), tiles = q4_tiles(a.dims);
    const size_t tile_bytes = (size_t)chunks * q4_chunk_bytes(GPC), plane = (size_t)a.pairs * a.width;
    const uint8_t* w = a.down + (size_t)e * a.down_bytes;
    const int term = (lane & 15) / PER;
    for (int m0 = 0; m0 < count; m0 += PER) {
        const uint16_t* row = nullptr;
        if (m0 + (lane & (PER - 1)) < count && term < TERMS)
            row = a.h + term * plane + (size_t)(m0 ? it.pair[m0 + (lane & (PER - 1))] : from) * a.width;
        const uint32_t mine = (blockIdx.x * WK + wave) * NT;
        if (mine < tiles) {
            const uint32_t tile0 = min(mine, tiles - NT);  // the last wave's tiles overlap
            f4v out[NT];
#pragma unroll
            for (int t = 0; t < NT; ++t) out[t] = f4v{0.0f, 0.0f, 0.0f, 0.0f};
            q4_stream<true, SBF, GPC, NT, NB, true>(w + tile0 * tile_bytes, tile_bytes, 0, 1, chunks, row, a.width, lane,
                                                  out);
            f4v v[NT];
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    v[t][i] = out[t][i];
                    if constexpr (TERMS == 3) v[t][i] = v[t][i] + lane_xor<16>(v[t][i]);
                    v[t][i] = v[t][i] + lane_xor<32>(v[t][i]);
                }
            q4_turn<NT>(turn[wave], v, lane, [&](int r, int c, const f4v& p) {
                if (r < PER && m0 + r < count)
                    *reinterpret_cast<f4v*>(a.y + (size_t)it.pair[m0 + r] * a.dims + tile0 * 16 + c) = p;
            });
        }
    }
}

// ---- the sums over groups of the activated values, for the biases of long items -------------------------------------------
__global__ void __launch_bounds__(256) q4_hsums_kernel(Q4MoeArgs a) {
    const uint32_t i = blockIdx.x * 4 + (threadIdx.x >> 6);
    if (i < a.pairs && (uint32_t)a.pick[i] < a.experts)
        q4_row_sums<true>(a.h + (size_t)i * a.width, a.terms, (size_t)a.pairs * a.width, a.width, a.group,
                          a.hsums + (size_t)i * q4_sum_bytes(a.width / a.group), threadIdx.x & 63, 0, 1);
}

// ---- long items -----------------------------------------------------------------------------------------------------
// An item's products by q4_gemm, with as many row groups as it has: NT4 tiles a wave with four of them, NT with fewer.
// Column blocks are counted in 4 NT4 tiles; the ones behind the last return. Rows of several terms are taken in two halves of
// the item: with four row groups down takes, at 2048 rows and with two terms, 250 us in place of 224 (groups of 64; 199 and 226
// with 32, 187 and 213 with 128, but 337 and 224 with fp16 scales, where registers run out), with three 505 in place of 260.
constexpr int q4_item_groups(int terms) { return terms > 1 ? 2 : 4; }
template <bool BF, bool SBF, int GPC, int NT4, int NT, int TERMS, bool RESIDENT, bool TURN, typename ROW, typename SUMS,
          typename STORE>
__device__ __forceinline__ void q4_item_gemm(uint8_t* lds, int count, const uint8_t* w, uint32_t tiles, uint32_t k,
                                             size_t plane, uint32_t cb, uint32_t cb_step, ROW row, SUMS sums, STORE store) {
    const auto go = [&](auto mt_, auto nt_, auto r, auto rs, auto st) __attribute__((always_inline)) {
        q4_gemm<BF, SBF, GPC, decltype(mt_)::value, decltype(nt_)::value, TERMS, RESIDENT, TURN>(lds, w, tiles, k, plane, cb,
                                                                                               cb_step, r, rs, st);
    };
    const std::integral_constant<int, 1> one;
    const std::integral_constant<int, 2> two;
    const std::integral_constant<int, NT> nt;
    if constexpr (q4_item_groups(TERMS) == 2) {
        static_assert(TURN && NT == NT4);
        for (int m0 = 0; m0 < count; m0 += 32) {
            const auto r = [&](int i) { return row(m0 + i); };
            const auto rs = [&](int i) { return sums(m0 + i); };
            const auto st = [&](int m, uint32_t col, const f4v& v) { store(m0 + m, col, v); };
            if (m0) __syncthreads();  // the first half's last readers of LDS
            if (count - m0 > 16) go(two, nt, r, rs, st);
            else go(one, nt, r, rs, st);
        }
    } else {
        if (count > 32) go(std::integral_constant<int, 4>{}, std::integral_constant<int, NT4>{}, row, sums, store);
        else if (cb * 4 * NT >= tiles) return;
        else if (count > 16) go(two, nt, row, sums, store);
        else go(one, nt, row, sums, store);
    }
}

// Blocks go to the card's eight dies in turn, and each die has an L2 of its own: die x takes the x-th eighth of the full items
// (of the partial ones), a run by expert, and all column blocks of its items, so that an expert's items share its weights on
// one die. Column blocks are the slow index: blocks behind an item's last one return at once, and where those come at a
// fixed distance they fall on the same shader engines, which leaves half of the card idle (gate|up, 256 rows: 167 against
// 96 us).
struct Q4Place {
    int item;  // -1: none
    uint32_t cb;
};
constexpr int Q4_DIES = 8;
__device__ __forceinline__ Q4Place q4_place(const Q4MoeArgs& a, uint32_t blocks) {
    const int n = a.nitems[0], full = a.nitems[1], rest = n - full;
    const int x = (int)(blockIdx.x % Q4_DIES);
    const uint32_t slot = blockIdx.x / Q4_DIES, each = gridDim.x / Q4_DIES / blocks, cb = slot / each;
    const int j = (int)(slot - cb * each);
    const int f0 = (int)((int64_t)full * x / Q4_DIES), f1 = (int)((int64_t)full * (x + 1) / Q4_DIES);
    const int r0 = (int)((int64_t)rest * x / Q4_DIES), r1 = (int)((int64_t)rest * (x + 1) / Q4_DIES);
    if (j < f1 - f0) return {f0 + j, cb};
    const int i = full + r0 + j - (f1 - f0);
    return {i < full + r1 ? i : -1, cb};
}
static unsigned q4_place_blocks(uint32_t max_items, uint32_t blocks) { return Q4_DIES * (max_items / Q4_DIES + 2) * blocks; }

// Two tiles a wave with more than 32 rows, else four: 2048 rows 265 us (390 TFLOP/s; 254 to 300 by the draw of the routing),
// with four throughout 290. Counters have the matrix units busy a fifth of the time and the vector units a third, with 1.4
// waves a SIMD on average of the two that the registers allow: waves wait for a chunk's rows, for each other and, at the end,
// for the last blocks. Items of up to 80 or 96 rows, which convert fewer weights, take as long (266, 280) at 2048 rows and
// longer (206, 218 against 185) at 1024; column blocks side by side in place of one after the other, for the rows' sake, 265 at
// 2048 and 228 at 1024. At 512 rows 256 experts just fill the card with two blocks each: 113 us, but 157 where one of them has
// 33 rows and four.
template <bool BF, bool SBF, int GPC, int NT4, int NT>
__global__ void __launch_bounds__(Q4_GEMM_THREADS, 2) q4_gateup_gemm_kernel(Q4MoeArgs a, uint32_t blocks) {
    __shared__ __attribute__((aligned(16))) uint8_t lds[q4_gemm_lds<4, 1>()];
    const Q4Place at = q4_place(a, blocks);
    if (at.item < 0) return;
    const Q4Item& it = a.items[at.item];
    const int e = it.expert, count = it.count;
    const auto row_of = [&](int i) { return (size_t)((uint32_t)it.pair[min(i, count - 1)] / a.slots); };
    q4_item_gemm<BF, SBF, GPC, NT4, NT, 1, false, false>(
        lds, count, a.gu + (size_t)e * a.gu_bytes, a.width / 8, a.dims, 0, at.cb, 1u << 24,
        [&](int i) { return a.x + row_of(i) * a.x_stride; },
        [&](int i) { return a.xsums + row_of(i) * q4_sum_bytes(a.dims / a.group); },
        [&](uint32_t tile, const auto& v) {
            const int lane = threadIdx.x & 63;
            const uint32_t col = tile * 8 + (lane & 7);
#pragma unroll
            for (int mt = 0; mt < (int)(sizeof(v) / sizeof(f4v)); ++mt)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float u = lane_xor<8>(v[mt][i]);  // lanes 0 .. 7 of 16 have the gate, the others the up column
                    const int m = 16 * mt + 4 * (lane >> 4) + i;
                    if ((lane & 8) || m >= count) continue;
                    store_terms(a.h, a.terms, (size_t)a.pairs * a.width, (size_t)it.pair[m] * a.width + col,
                                swiglu(v[mt][i], u));
                }
        });
}

// A block takes every `blocks`-th column block of an item, six blocks an item at most, and with RESIDENT keeps its rows in LDS
// meanwhile. 2048 rows 224 us with two terms, 249 with three: 403 MB of fp32 sums written and 226 MB of weights read. With a
// weight turned into an operand once a term in place of once, two terms took 323 us and three 345.
template <bool SBF, int GPC, int TERMS, int NT, bool RESIDENT>
__global__ void __launch_bounds__(Q4_GEMM_THREADS, 2) q4_down_gemm_kernel(Q4MoeArgs a, uint32_t blocks) {
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    const Q4Place at = q4_place(a, blocks);
    if (at.item < 0) return;
    const Q4Item& it = a.items[at.item];
    const int e = it.expert, count = it.count;
    q4_item_gemm<true, SBF, GPC, NT, NT, TERMS, RESIDENT, true>(
        lds, count, a.down + (size_t)e * a.down_bytes, q4_tiles(a.dims), a.width, (size_t)a.pairs * a.width, at.cb, blocks,
        [&](int i) { return a.h + (size_t)it.pair[min(i, count - 1)] * a.width; },
        [&](int i) { return a.hsums + (size_t)it.pair[min(i, count - 1)] * q4_sum_bytes(a.width / a.group); },
        [&](int m, uint32_t col, const f4v& v) {
            if (m < count) *reinterpret_cast<f4v*>(a.y + (size_t)it.pair[m] * a.dims + col) = v;
        });
}

// ---- a row's slots, in order ----------------------------------------------------------------------------------------
// Bound by the pairs' sums: 64 rows 6.5 us (12.6 MB), 2048 rows 94 us (403 MB read, 25 MB written: 4.6 TB/s).
__global__ void __launch_bounds__(256) q4_combine_kernel(Q4MoeArgs a) {
    __shared__ int32_t pick[32];
    __shared__ float weight[32];
    const uint32_t r = blockIdx.x, d = (blockIdx.y * 256 + threadIdx.x) * 4;
    if (threadIdx.x < a.slots) pick[threadIdx.x] = a.pick[(size_t)r * a.slots + threadIdx.x];
    __syncthreads();
    if (threadIdx.x < a.slots) {  // an expert named again adds its weight to the first naming
        const int32_t e = pick[threadIdx.x];
        bool first = (uint32_t)e < a.experts;
        float w = 0.0f;
        for (uint32_t k = 0; k < a.slots; ++k) {
            first = first && !(k < threadIdx.x && pick[k] == e);
            if (k >= threadIdx.x && pick[k] == e) w = w + a.wts[(size_t)r * a.slots + k];
        }
        weight[threadIdx.x] = w;
        __builtin_amdgcn_wave_barrier();
        if (!first) pick[threadIdx.x] = -1;
    }
    __syncthreads();
    if (d >= a.dims) return;
    f4v v{0.0f, 0.0f, 0.0f, 0.0f};
    const float* y = a.y + (size_t)r * a.slots * a.dims + d;
    for (uint32_t k0 = 0; k0 < a.slots; k0 += 8) {  // eight slots' loads at once; what is no expert's is not used
        f4v p[8];
        bool has[8];
#pragma unroll
        for (uint32_t k = 0; k < 8; ++k) {
            has[k] = k0 + k < a.slots && pick[k0 + k] >= 0;
            p[k] = *reinterpret_cast<const f4v*>(y + (size_t)min(k0 + k, a.slots - 1) * a.dims);
        }
#pragma unroll
        for (uint32_t k = 0; k < 8; ++k)
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = has[k] ? __builtin_fmaf(weight[k0 + k], p[k][i], v[i]) : v[i];
    }
    const size_t at = (size_t)r * a.dims + d;
    if (a.out_dtype == F32) {
        typedef f4v f4v_a4 __attribute__((aligned(4)));
        *reinterpret_cast<f4v_a4*>(static_cast<float*>(a.out) + at) = v;
    } else {
        typedef u2v u2v_a2 __attribute__((aligned(2)));
        uint16_t b[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) b[i] = a.out_dtype == BF16 ? f2bf(v[i]) : f2h(v[i]);
        *reinterpret_cast<u2v_a2*>(static_cast<uint16_t*>(a.out) + at) =
            u2v{(uint32_t)b[0] | (uint32_t)b[1] << 16, (uint32_t)b[2] | (uint32_t)b[3] << 16};
    }
}

// ---- launches -------------------------------------------------------------------------------------------------------
static void launch_gateup(hipStream_t s, const Q4MoeArgs& a, bool bf, bool sbf, int gpc, uint32_t max_items) {
    const uint32_t tiles = a.width / 8;
    q4_types(bf, sbf, gpc, [&](auto gpc_, auto bf_, auto sbf_) {
        constexpr bool BF = decltype(bf_)::value, SBF = decltype(sbf_)::value;
        constexpr int GPC = decltype(gpc_)::value;
        if (a.rows == 1) q4_gateup_kernel<BF, SBF, GPC, 1, 8, 3, ONE_ROW><<<dim3(tiles, a.pairs), 512, 0, s>>>(a);
        else if (a.rows <= Q4_ROWS)
            q4_gateup_kernel<BF, SBF, GPC, 2, 8, 3, FEW_ROWS><<<dim3(tiles / 2, a.pairs + 1), 512, 0, s>>>(a);
        else if (a.item == Q4_BIG_ITEM) {
            const uint32_t blocks = (tiles + 7) / 8;
            const unsigned grid = q4_place_blocks(max_items, blocks);
            q4_gateup_gemm_kernel<BF, SBF, GPC, 2, 4><<<grid, Q4_GEMM_THREADS, 0, s>>>(a, blocks);
        } else q4_gateup_kernel<BF, SBF, GPC, 2, 8, 3, ITEMS><<<dim3(tiles / 2, max_items), 512, 0, s>>>(a);
    });
}

template <int TERMS>
static void launch_down(hipStream_t s, const Q4MoeArgs& a, bool sbf, int gpc, uint32_t max_items) {
    const uint32_t tiles = q4_tiles(a.dims);
    q4_types(true, sbf, gpc, [&](auto gpc_, auto bf_, auto sbf_) {
        if constexpr (decltype(bf_)::value) {
            constexpr bool SBF = decltype(sbf_)::value;
            constexpr int GPC = decltype(gpc_)::value;
            if (a.rows == 1) q4_down_one_kernel<SBF, GPC, TERMS, 1, 8, 2><<<tiles, 512, 0, s>>>(a);
            else if (a.item == Q4_BIG_ITEM) {
                constexpr int MT = q4_item_groups(TERMS), NT = 4;
                const uint32_t chunks = q4_chunks(a.width);
                const auto blocks = [&](uint32_t nt) { return std::min((tiles + 4 * nt - 1) / (4 * nt), 6u); };
                if (chunks <= Q4_RESIDENT / (TERMS * MT * 4096))
                    q4_down_gemm_kernel<SBF, GPC, TERMS, 4, true>
                        <<<q4_place_blocks(max_items, blocks(4)), Q4_GEMM_THREADS,
                           q4_gemm_lds<MT, TERMS>((int)chunks, (int)(chunks * GPC + 7) / 8), s>>>(a, blocks(4));
                else
                    q4_down_gemm_kernel<SBF, GPC, TERMS, NT, false>
                        <<<q4_place_blocks(max_items, blocks(NT)), Q4_GEMM_THREADS, q4_gemm_lds<MT, TERMS>(), s>>>(a, blocks(NT));
            } else if (tiles >= 4) q4_down_kernel<SBF, GPC, TERMS, 4, 8, 1><<<dim3((tiles + 31) / 32, max_items), 512, 0, s>>>(a);
            else q4_down_kernel<SBF, GPC, TERMS, 1, 4, 1><<<dim3((tiles + 3) / 4, max_items), 256, 0, s>>>(a);
        }
    });
}

// Terms of the activated values: more bits than the output's type can show (bf16 8, fp16 11, fp32 24), so that the output's
// own rounding is what its error comes from. One term with bf16 out was off by 0.0023 of the output's norm where its rounding
// is 0.0017, for 0.4 to 1.6 us less of down up to 64 rows and 195 in place of 265 us at 2048.
static int q4_terms(int out_dtype) { return out_dtype == F32 ? 3 : 2; }

static uint32_t q4_max_items(uint32_t experts, size_t pairs, uint32_t item = Q4_ITEM) {
    const size_t full = pairs / item, some = pairs < experts ? pairs : experts;
    return (uint32_t)(full + some);
}

static int q4_experts_ok(const ea_q4_experts* ex) {
    if (!ex || !ex->gu || !ex->down || ((ex->gu | ex->down) & 15)) return EA_BAD_ARGUMENT;
    if (ex->s_dtype != F16 && ex->s_dtype != BF16) return EA_BAD_ARGUMENT;
    if (ex->group != 32 && ex->group != 64 && ex->group != 128) return EA_BAD_WIDTH;
    if (ex->count == 0 || ex->dims == 0 || ex->width == 0) return EA_BAD_ARGUMENT;
    if (ex->count > Q4_MAX_EXPERTS) return EA_TOO_MANY_EXPERTS;
    if (ex->dims % ex->group != 0 || ex->width % ex->group != 0) return EA_UNEVEN_SPLIT;
    return EA_OK;
}

static size_t up256(size_t n) { return (n + 255) & ~(size_t)255; }

// Carves a scratch; returns its bytes (base 0: the size alone).
static size_t q4_carve(ea_q4_scratch* s, uint64_t base, const ea_q4_experts* ex, uint32_t rows, uint32_t slots) {
    const size_t pairs = (size_t)rows * slots;
    size_t at = 0;
    auto take = [&](size_t bytes) {
        const uint64_t p = base + at;
        at += up256(bytes);
        return p;
    };
    s->items = take(sizeof(Q4Item) * q4_max_items(ex->count, pairs));
    s->count = take(8);
    s->h = take(3 * 2 * pairs * ex->width);
    s->y = take(4 * (size_t)pairs * ex->dims);
    s->sums = take((size_t)rows * q4_sum_bytes(ex->dims / 32) + 64);
    s->hsums = take(pairs * q4_sum_bytes(ex->width / 32) + 64);
    s->rows = rows;
    s->slots = slots;
    return at;
}

}  // namespace ea

using namespace ea;

extern "C" {

size_t ea_q4_scratch_bytes(const ea_q4_experts* ex, uint32_t rows, uint32_t slots) {
    ea_q4_scratch s;
    if (q4_experts_ok(ex) || rows == 0 || slots == 0 || slots > 32 || (uint64_t)rows * slots > EA_Q4_MAX_PAIRS) return 0;
    return q4_carve(&s, 0, ex, rows, slots);
}

int ea_q4_scratch_init(ea_q4_scratch* s, void* base, size_t bytes, const ea_q4_experts* ex, uint32_t rows,
                       uint32_t slots) {
    int r = q4_experts_ok(ex);
    if (r) return r;
    if (!s || !base || (reinterpret_cast<uintptr_t>(base) & 255) || rows == 0) return EA_BAD_ARGUMENT;
    if (slots == 0 || slots > 32) return EA_TOO_MANY_SLOTS;
    if ((uint64_t)rows * slots > EA_Q4_MAX_PAIRS) return EA_BAD_ARGUMENT;
    if (bytes < ea_q4_scratch_bytes(ex, rows, slots)) return EA_SCRATCH_TOO_SMALL;
    q4_carve(s, (uint64_t)reinterpret_cast<uintptr_t>(base), ex, rows, slots);
    s->experts = ex->count;
    s->dims = ex->dims;
    s->width = ex->width;
    return EA_OK;
}

int ea_q4_routed(ea_stream_t stream, const void* x, int x_dtype, uint32_t x_stride, const int32_t* pick, const float* wts,
                 const ea_q4_experts* ex, const ea_q4_scratch* sc, void* out, int out_dtype, uint32_t R) {
    int r = q4_experts_ok(ex);
    if (r) return r;
    if (!x || !pick || !wts || !sc || !out || !sc->y) return EA_BAD_ARGUMENT;
    if ((x_dtype != F16 && x_dtype != BF16) || out_dtype < F16 || out_dtype > F32) return EA_BAD_ARGUMENT;
    if (reinterpret_cast<uintptr_t>(x) & 7) return EA_BAD_ARGUMENT;
    if (x_stride < ex->dims || x_stride % 4 != 0) return EA_BAD_ROW_STRIDE;
    if (R > sc->rows || ex->count > sc->experts || ex->dims > sc->dims || ex->width > sc->width) return EA_SCRATCH_TOO_SMALL;
    EA_REQUIRE_CTX(ctx_);
    (void)ctx_;
    if (R == 0) return EA_OK;
    const int gpc = 128 / (int)ex->group;
    Q4MoeArgs a{};
    a.x = static_cast<const uint16_t*>(x);
    a.x_stride = x_stride;
    a.pick = pick;
    a.wts = wts;
    a.gu = dptr<const uint8_t>(ex->gu);
    a.down = dptr<const uint8_t>(ex->down);
    a.gu_bytes = (size_t)(ex->width / 8) * q4_chunks(ex->dims) * q4_chunk_bytes(gpc);
    a.down_bytes = (size_t)q4_tiles(ex->dims) * q4_chunks(ex->width) * q4_chunk_bytes(gpc);
    a.nitems = dptr<int32_t>(sc->count);
    a.items = dptr<Q4Item>(sc->items);
    a.h = dptr<uint16_t>(sc->h);
    a.y = dptr<float>(sc->y);
    a.xsums = dptr<uint8_t>(sc->sums);
    a.hsums = dptr<uint8_t>(sc->hsums);
    a.group = ex->group;
    a.bf = x_dtype == BF16;
    a.out = out;
    a.rows = R;
    a.pairs = R * sc->slots;
    a.dims = ex->dims;
    a.width = ex->width;
    a.experts = ex->count;
    a.slots = sc->slots;
    a.out_dtype = out_dtype;
    a.terms = q4_terms(out_dtype);
    // Long items pay where experts have more than about seven rows each (down's short items turn a weight once for every eight
    // rows of two terms, or four of three) and where there are blocks enough to fill the card, as an item's waves no longer share
    // a tile's chunks. All launches with short / long items, bf16 out: 128 rows 162 / 174 us, 256 201 / 187, 320 226 / 201, 384
    // 252 / 212, 512 320 / 229, 2048 960 / 598; fp32 out: 320 265 / 208, 2048 1196 / 614.
    const uint64_t some = std::min<uint64_t>(a.pairs, a.experts), column_blocks = (a.width / 8 + 7) / 8;
    const bool big = R > Q4_ROWS && a.pairs > 7 * some && (a.pairs / Q4_BIG_ITEM + some / 2) * column_blocks >= 512;
    a.item = big ? Q4_BIG_ITEM : Q4_ITEM;
    const uint32_t max_items = q4_max_items(a.experts, a.pairs, a.item);
    hipStream_t s = as_stream(stream);
    const bool sbf = ex->s_dtype == BF16;
    if (R > Q4_ROWS) q4_group_kernel<<<1 + (big ? (R * Q4_SUM_WAVES + 15) / 16 : 0), 1024, 0, s>>>(a);
    launch_gateup(s, a, x_dtype == BF16, sbf, gpc, max_items);
    if (big) q4_hsums_kernel<<<(a.pairs + 3) / 4, 256, 0, s>>>(a);
    if (a.terms == 2) launch_down<2>(s, a, sbf, gpc, max_items);
    else launch_down<3>(s, a, sbf, gpc, max_items);
    if (R > 1) q4_combine_kernel<<<dim3(R, (a.dims + 1023) / 1024), 256, 0, s>>>(a);
    return launched();
}

}  // extern "C"
