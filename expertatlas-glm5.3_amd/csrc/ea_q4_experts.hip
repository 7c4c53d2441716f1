// Routed experts with 4-bit weights in groups: out[r] = sum over slots of wts * down_e(silu(gate_e x) * (up_e x)).
//
// The rows' picks are sorted by expert and cut into items (an expert and up to 16 of its pairs); a block multiplies an
// item's rows by tiles of the expert's gate|up (8 columns of each) and writes the activated pairs; another multiplies those
// by tiles of the down projection; the last launch adds a row's slots in order. A pair's values depend neither on the others
// of its item nor on their order, so the results are the same on every run.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "ea_host.hpp"
#include "ea_q4.hpp"

namespace ea {

constexpr uint32_t Q4_MAX_EXPERTS = 4096;
constexpr uint32_t Q4_ITEM = 16;                       // rows an item
constexpr uint32_t Q4_ROWS = 16, Q4_PAIRS = Q4_ROWS * 32;  // rows and pairs that are grouped beside the first products

struct Q4Item {
    int32_t expert, first, count, pad;
};

struct Q4MoeArgs {
    const uint16_t* x;
    size_t x_stride;
    const int32_t* pick;
    const float* wts;
    const uint8_t *gu, *down;
    size_t gu_bytes, down_bytes;  // one expert's
    int32_t *sorted, *nitems;     // pairs by expert; the number of items
    Q4Item* items;                // runs of sorted
    uint16_t* h;                  // bf16 [terms][pairs][width]
    float* y;                     // fp32 [pairs][dims]
    void* out;
    uint32_t rows, pairs, dims, width, experts, slots;
    int out_dtype;
    bool sbf;
};

// ---- grouping -----------------------------------------------------------------------------------------------------
// One block: the pairs of each expert counted, the counts scanned, the pairs placed (in any order within an expert), the
// items listed. A pick outside 0 .. experts - 1 is a slot without an expert.
__global__ void __launch_bounds__(1024) q4_group_kernel(Q4MoeArgs a) {
    __shared__ uint32_t count[Q4_MAX_EXPERTS], start[Q4_MAX_EXPERTS], sums[2][16];
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    for (uint32_t e = t; e < a.experts; e += 1024) count[e] = 0;
    __syncthreads();
    for (uint32_t p = t; p < a.pairs; p += 1024) {
        const uint32_t e = (uint32_t)a.pick[p];
        if (e < a.experts) atomicAdd(&count[e], 1u);
    }
    __syncthreads();
    // exclusive scans of the counts and the item counts, 1024 experts a step
    uint32_t base = 0, ibase = 0;
    for (uint32_t e0 = 0; e0 < a.experts; e0 += 1024) {
        const uint32_t e = e0 + t, c = e < a.experts ? count[e] : 0, n = (c + Q4_ITEM - 1) / Q4_ITEM;
        uint32_t v = c, w = n;
        for (int d = 1; d < 64; d <<= 1) {
            const uint32_t pv = __shfl_up(v, d), pw = __shfl_up(w, d);
            if (lane >= d) v += pv, w += pw;
        }
        if (lane == 63) sums[0][wave] = v, sums[1][wave] = w;
        __syncthreads();
        uint32_t bv = base, bw = ibase;
        for (int i = 0; i < 16; ++i) {
            const uint32_t sv = sums[0][i], sw = sums[1][i];
            if (i < wave) bv += sv, bw += sw;
            base += sv;
            ibase += sw;
        }
        const uint32_t first = bv + v - c, item = bw + w - n;
        if (e < a.experts) start[e] = first;
        for (uint32_t i = 0; i < n; ++i)
            a.items[item + i] = Q4Item{(int32_t)e, (int32_t)(first + i * Q4_ITEM), (int32_t)min(c - i * Q4_ITEM, Q4_ITEM), 0};
        __syncthreads();
    }
    if (t == 0) *a.nitems = (int32_t)ibase;
    for (uint32_t p = t; p < a.pairs; p += 1024) {
        const uint32_t e = (uint32_t)a.pick[p];
        if (e < a.experts) a.sorted[atomicAdd(&start[e], 1u)] = (int32_t)p;
    }
}

// The same for up to 16 rows, in the order of the experts' first pairs, by a block beside the first products (picks: the
// call's, in LDS, changed). An expert is one item, and a row that names it again is left out: the last launch gives its
// weight to the first naming.
template <int THREADS>
__device__ void q4_group_rows(const Q4MoeArgs& a, int32_t* picks) {
    __shared__ int16_t owner[Q4_PAIRS], before[Q4_PAIRS], count[Q4_PAIRS], first[Q4_PAIRS];
    int32_t once[(Q4_PAIRS + THREADS - 1) / THREADS];
    for (uint32_t p = threadIdx.x, i = 0; p < a.pairs; p += THREADS, ++i) {
        int32_t e = picks[p];
        e = (uint32_t)e < a.experts ? e : -1;
        for (uint32_t q = p - p % a.slots; q < p; ++q) e = picks[q] == e ? -1 : e;
        once[i] = e;
        count[p] = 0;
    }
    __syncthreads();
    for (uint32_t p = threadIdx.x, i = 0; p < a.pairs; p += THREADS, ++i) picks[p] = once[i];
    __syncthreads();
    for (uint32_t p = threadIdx.x; p < a.pairs; p += THREADS) {
        const int32_t e = picks[p];
        uint32_t n = 0, own = p, all = 0;
        if (e >= 0) {
#pragma unroll 4
            for (uint32_t q = 0; q < a.pairs; ++q) {
                const bool same = picks[q] == e;
                own = same && all == 0 ? q : own;
                n += same && q < p;
                all += same;
            }
        }
        owner[p] = (int16_t)own;
        before[p] = e >= 0 ? (int16_t)n : -1;
        count[p] = (int16_t)all;
    }
    __syncthreads();
    if (threadIdx.x < 64) {
        int items = 0, at = 0;
        for (uint32_t p0 = 0; p0 < a.pairs; p0 += 64) {
            const uint32_t p = p0 + threadIdx.x;
            const bool fresh = p < a.pairs && before[p] == 0;
            const int c = fresh ? count[p] : 0;
            int sum = c;
            for (int d = 1; d < 64; d <<= 1) {
                const int o = __shfl_up(sum, d);
                sum += (int)threadIdx.x >= d ? o : 0;
            }
            const uint64_t all = __ballot(fresh);
            if (fresh) {
                first[p] = (int16_t)(at + sum - c);
                a.items[items + __builtin_popcountll(all & ((1ull << threadIdx.x) - 1))] = Q4Item{picks[p], at + sum - c, c, 0};
            }
            items += __builtin_popcountll(all);
            at += __shfl(sum, 63);
        }
        if (threadIdx.x == 0) *a.nitems = items;
    }
    __syncthreads();
    for (uint32_t p = threadIdx.x; p < a.pairs; p += THREADS)
        if (before[p] >= 0) a.sorted[first[owner[p]] + before[p]] = (int32_t)p;
}

__device__ __forceinline__ float swiglu(float g, float u) { return g / (1.0f + expf_path(0.0f - g)) * u; }

// An activated value as TERMS bf16 numbers that add up to it (8 bits each).
template <int TERMS>
__device__ __forceinline__ void store_terms(uint16_t* h, size_t plane, size_t at, float v) {
#pragma unroll
    for (int i = 0; i < TERMS; ++i) {
        const uint16_t b = f2bf(v);
        h[(size_t)i * plane + at] = b;
        v = __builtin_fabsf(v) < __builtin_inff() ? v - bf2f(b) : 0.0f;
    }
}

// ---- gate | up ------------------------------------------------------------------------------------------------------
// Block (NT tiles of gate | up, item): 16 rows of a matrix instruction, those that the item does not have as zeros, which
// cost neither loads nor cache; WK waves take every WK-th chunk. Up to 16 rows nothing is sorted before: block (tiles, pair)
// works if no earlier pair names its expert, a row of the instruction is the row of x, and one more block groups the pairs
// for the launches behind.
enum Q4Rows { ONE_ROW, FEW_ROWS, ITEMS };

template <bool BF, int GPC, int TERMS, int NT, int WK, int NB, int MODE>
__global__ void __launch_bounds__(64 * WK) q4_gateup_kernel(Q4MoeArgs a) {
    __shared__ f4v part[WK][NT][1][64];
    __shared__ int32_t picks[MODE == FEW_ROWS ? Q4_PAIRS : 16];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t u = blockIdx.y, chunks = q4_chunks(a.dims), tiles = (a.width + 7) / 8, r = lane & 15;
    int32_t e;
    const uint16_t* row[1] = {nullptr};
    Q4Item it{};
    if constexpr (MODE == ONE_ROW) {  // every slot by itself: nothing is compared before the weights are read
        e = a.pick[u];
        if ((uint32_t)e >= a.experts) return;
        if (r == 0) row[0] = a.x;
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
                if (picks[r * a.slots + k] == e) row[0] = a.x + (size_t)r * a.x_stride;
    } else {
        if ((int)u >= *a.nitems) return;
        it = a.items[u];
        e = it.expert;
        const int32_t p = a.sorted[it.first + min((int)r, it.count - 1)];
        if (threadIdx.x < 16) picks[r] = p;
        if ((int)r < it.count) row[0] = a.x + (size_t)((uint32_t)p / a.slots) * a.x_stride;
    }
    const uint32_t tile0 = min(blockIdx.x * NT, tiles - NT);  // the last block's tiles overlap
    const size_t tile_bytes = (size_t)chunks * q4_chunk_bytes(GPC);
    f4v out[NT][1];
#pragma unroll
    for (int t = 0; t < NT; ++t) out[t][0] = f4v{0.0f, 0.0f, 0.0f, 0.0f};
    q4_stream<BF, GPC, 1, NT, NB, true>(a.gu + (size_t)e * a.gu_bytes + tile0 * tile_bytes, tile_bytes, wave, WK, chunks, row,
                                        a.dims, lane, a.sbf, out);
#pragma unroll
    for (int t = 0; t < NT; ++t) part[wave][t][0][lane] = out[t][0];
    __syncthreads();
    for (int i = threadIdx.x; i < 128 * NT; i += 64 * WK) {
        const int n = i & 7, t = (i >> 3) % NT, m = i / (8 * NT);
        const uint32_t col = (tile0 + t) * 8 + n;
        uint32_t p = u;
        bool is = col < a.width;
        if constexpr (MODE == ONE_ROW) is = is && m == 0;
        if constexpr (MODE == FEW_ROWS) {  // the row's first naming of the expert
            p = m * a.slots;
            const uint32_t end = (uint32_t)m < a.rows ? p + a.slots : p;
            while (p < end && picks[p] != e) ++p;
            is = is && p < end;
        }
        if constexpr (MODE == ITEMS) {
            p = picks[m];
            is = is && m < it.count;
        }
        if (!is) continue;
        const float v = swiglu(q4_total<WK, NT, 1>(part, t, 0, m, n), q4_total<WK, NT, 1>(part, t, 0, m, n + 8));
        store_terms<TERMS>(a.h, (size_t)a.pairs * a.width, (size_t)p * a.width + col, v);
    }
}

// ---- down -----------------------------------------------------------------------------------------------------------
// One row: NT tiles of the output a block; its waves take the (slot, chunk) units in turn, weigh their sums in registers, and
// terms (rows 0 .. TERMS - 1 of the instruction) and waves are added at the end.
template <int GPC, int TERMS, int NT, int WK, int NB>
__global__ void __launch_bounds__(64 * WK) q4_down_one_kernel(Q4MoeArgs a) {
    __shared__ f4v part[WK][NT][1][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), term = lane & 15;
    const uint32_t chunks = q4_chunks(a.width), tiles = q4_tiles(a.dims), units = a.slots * chunks;
    const uint32_t tile0 = min(blockIdx.x * NT, tiles - NT);
    const size_t tile_bytes = (size_t)chunks * q4_chunk_bytes(GPC), plane = (size_t)a.slots * a.width;
    f4v out[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) out[t] = f4v{0.0f, 0.0f, 0.0f, 0.0f};
    for (uint32_t u0 = wave; u0 < units; u0 += WK * NB) {
        u4v words[NB][NT], x[NB][1][4];
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
            for (int j = 0; j < 4; ++j) x[i][0][j] = u4v{0, 0, 0, 0};
        if (term < TERMS) {
#pragma unroll
            for (int i = 0; i < NB; ++i) {
                const uint32_t u = min(u0 + WK * i, units - 1);
                q4_rows(a.h + term * plane + (size_t)(u / chunks) * a.width, u % chunks, a.width, lane, x[i][0]);
            }
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < NB; ++i) {
            if (u0 + WK * i >= units || (uint32_t)e[i] >= a.experts) continue;
            f4v y[NT][1];
#pragma unroll
            for (int t = 0; t < NT; ++t) y[t][0] = f4v{0.0f, 0.0f, 0.0f, 0.0f};
            q4_chunk<true, GPC, 1, NT>(words[i], par[i], x[i], a.sbf, y);
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int r = 0; r < TERMS; ++r) out[t][r] = __builtin_fmaf(w[i], y[t][0][r], out[t][r]);
        }
    }
#pragma unroll
    for (int t = 0; t < NT; ++t) part[wave][t][0][lane] = out[t];
    __syncthreads();
    for (int i = threadIdx.x; i < 16 * NT; i += 64 * WK) {
        const int n = i & 15, t = i >> 4;
        const uint32_t col = (tile0 + t) * 16 + n;
        if (col >= a.dims) continue;
        float v = q4_total<WK, NT, 1>(part, t, 0, TERMS - 1, n);
#pragma unroll
        for (int r = TERMS - 2; r >= 0; --r) v = v + q4_total<WK, NT, 1>(part, t, 0, r, n);  // the small terms first
        store_act(a.out, a.out_dtype, col, v);
    }
}

// More rows: block (WK NT tiles, item), a wave its NT tiles over all of the width, so that no sum crosses waves and an
// expert's weights are read where they lie together (blocks that took some tiles of every expert read them at half the rate).
// Terms are rows of their own: rows 4 q .. 4 q + 3 of the instruction are quad q of the accumulators' lanes; with three
// terms quad q holds term q of four pairs, with two quads 2 q and 2 q + 1 term q of eight, and adding lanes 16 (and 32)
// apart adds the terms.
template <int GPC, int TERMS, int NT, int WK, int NB>
__global__ void __launch_bounds__(64 * WK) q4_down_kernel(Q4MoeArgs a) {
    constexpr int PER = TERMS == 1 ? 16 : TERMS == 2 ? 8 : 4;  // pairs a product
    if ((int)blockIdx.y >= *a.nitems) return;
    const Q4Item it = a.items[blockIdx.y];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t chunks = q4_chunks(a.width), tiles = q4_tiles(a.dims), mine = (blockIdx.x * WK + wave) * NT;
    if (mine >= tiles) return;
    const uint32_t tile0 = min(mine, tiles - NT);  // the last wave's tiles overlap
    const size_t tile_bytes = (size_t)chunks * q4_chunk_bytes(GPC), plane = (size_t)a.pairs * a.width;
    const uint8_t* w = a.down + (size_t)it.expert * a.down_bytes + tile0 * tile_bytes;
    for (int m0 = 0; m0 < it.count; m0 += PER) {
        const int m = m0 + (lane & (PER - 1)), term = (lane & 15) / PER;
        const uint16_t* row[1] = {nullptr};
        if (m < it.count && term < TERMS) row[0] = a.h + term * plane + (size_t)a.sorted[it.first + m] * a.width;
        f4v out[NT][1];
#pragma unroll
        for (int t = 0; t < NT; ++t) out[t][0] = f4v{0.0f, 0.0f, 0.0f, 0.0f};
        q4_stream<true, GPC, 1, NT, NB, true>(w, tile_bytes, 0, 1, chunks, row, a.width, lane, a.sbf, out);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int q = lane >> 4, at = m0 + 4 * (q & (PER / 4 - 1)) + i;  // the pair of this quad's value i
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                float v = out[t][0][i];
                if constexpr (TERMS == 3) v = v + lane_xor<16>(v);
                if constexpr (TERMS >= 2) v = v + lane_xor<32>(v);
                const uint32_t col = (tile0 + t) * 16 + (lane & 15);
                if (at < it.count && q < PER / 4 && col < a.dims)
                    a.y[(size_t)a.sorted[it.first + at] * a.dims + col] = v;
            }
        }
    }
}

// ---- a row's slots, in order ----------------------------------------------------------------------------------------
__global__ void __launch_bounds__(256) q4_combine_kernel(Q4MoeArgs a) {
    __shared__ int32_t pick[32];
    __shared__ float weight[32];
    const uint32_t r = blockIdx.x, d = blockIdx.y * 256 + threadIdx.x;
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
    float v = 0.0f;
    for (uint32_t k = 0; k < a.slots; ++k)
        if (pick[k] >= 0) v = __builtin_fmaf(weight[k], a.y[((size_t)r * a.slots + k) * a.dims + d], v);
    store_act(a.out, a.out_dtype, (size_t)r * a.dims + d, v);
}

// ---- launches -------------------------------------------------------------------------------------------------------
template <int GPC, int TERMS>
static void launch_moe(hipStream_t s, const Q4MoeArgs& a, bool bf, uint32_t max_items) {
    const uint32_t tiles = (a.width + 7) / 8, dtiles = q4_tiles(a.dims);
    auto gateup = [&](auto bf_, auto nt_, auto mode_, uint32_t blocks) {
        constexpr int NT = decltype(nt_)::value, WK = 8;
        q4_gateup_kernel<decltype(bf_)::value, GPC, TERMS, NT, WK, 3, decltype(mode_)::value>
            <<<dim3((tiles + NT - 1) / NT, blocks), 64 * WK, 0, s>>>(a);
    };
    auto with = [&](auto nt_, auto mode_, uint32_t blocks) {
        if (bf) gateup(std::true_type{}, nt_, mode_, blocks);
        else gateup(std::false_type{}, nt_, mode_, blocks);
    };
    using One = std::integral_constant<int, 1>;
    using Two = std::integral_constant<int, 2>;
    if (a.rows == 1) {
        with(One{}, std::integral_constant<int, ONE_ROW>{}, a.pairs);
        q4_down_one_kernel<GPC, TERMS, 1, 8, 2><<<dtiles, 512, 0, s>>>(a);
        return;
    }
    if (a.rows <= Q4_ROWS) {
        const std::integral_constant<int, FEW_ROWS> few{};
        if (a.rows <= 4 || tiles < 2) with(One{}, few, a.pairs + 1);
        else with(Two{}, few, a.pairs + 1);
    } else {
        q4_group_kernel<<<1, 1024, 0, s>>>(a);
        const std::integral_constant<int, ITEMS> items{};
        if (tiles < 2) with(One{}, items, max_items);
        else with(Two{}, items, max_items);
    }
    if (dtiles >= 4) q4_down_kernel<GPC, TERMS, 4, 4, 2><<<dim3((dtiles + 15) / 16, max_items), 256, 0, s>>>(a);
    else q4_down_kernel<GPC, TERMS, 1, 4, 2><<<dim3((dtiles + 3) / 4, max_items), 256, 0, s>>>(a);
    q4_combine_kernel<<<dim3(a.rows, (a.dims + 255) / 256), 256, 0, s>>>(a);
}

// Terms of the activated values: what the output's type can show (bf16 8 bits, fp16 11, fp32 24).
static int q4_terms(int out_dtype) { return out_dtype == BF16 ? 1 : out_dtype == F16 ? 2 : 3; }

static uint32_t q4_max_items(uint32_t experts, size_t pairs) {
    const size_t full = pairs / Q4_ITEM, some = pairs < experts ? pairs : experts;
    return (uint32_t)(full + some);
}

static int q4_experts_ok(const ea_q4_experts* ex) {
    if (!ex || !ex->gu || !ex->down || (ex->s_dtype != F16 && ex->s_dtype != BF16)) return EA_BAD_ARGUMENT;
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
    s->sorted = take(4 * pairs);
    s->items = take(sizeof(Q4Item) * q4_max_items(ex->count, pairs));
    s->count = take(4);
    s->h = take(3 * 2 * pairs * ex->width);
    s->y = take(4 * pairs * ex->dims);
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
    const int gpc = 128 / (int)ex->group, terms = q4_terms(out_dtype);
    Q4MoeArgs a{};
    a.x = static_cast<const uint16_t*>(x);
    a.x_stride = x_stride;
    a.pick = pick;
    a.wts = wts;
    a.gu = dptr<const uint8_t>(ex->gu);
    a.down = dptr<const uint8_t>(ex->down);
    a.gu_bytes = (size_t)((ex->width + 7) / 8) * q4_chunks(ex->dims) * q4_chunk_bytes(gpc);
    a.down_bytes = (size_t)q4_tiles(ex->dims) * q4_chunks(ex->width) * q4_chunk_bytes(gpc);
    a.sorted = dptr<int32_t>(sc->sorted);
    a.nitems = dptr<int32_t>(sc->count);
    a.items = dptr<Q4Item>(sc->items);
    a.h = dptr<uint16_t>(sc->h);
    a.y = dptr<float>(sc->y);
    a.out = out;
    a.rows = R;
    a.pairs = R * sc->slots;
    a.dims = ex->dims;
    a.width = ex->width;
    a.experts = ex->count;
    a.slots = sc->slots;
    a.out_dtype = out_dtype;
    a.sbf = ex->s_dtype == BF16;
    const uint32_t max_items = q4_max_items(a.experts, a.pairs);
    hipStream_t s = as_stream(stream);
    auto go = [&](auto gpc_) {
        constexpr int GPC = decltype(gpc_)::value;
        if (terms == 1) launch_moe<GPC, 1>(s, a, x_dtype == BF16, max_items);
        else if (terms == 2) launch_moe<GPC, 2>(s, a, x_dtype == BF16, max_items);
        else launch_moe<GPC, 3>(s, a, x_dtype == BF16, max_items);
    };
    if (gpc == 4) go(std::integral_constant<int, 4>{});
    else if (gpc == 2) go(std::integral_constant<int, 2>{});
    else go(std::integral_constant<int, 1>{});
    return launched();
}

}  // extern "C"
