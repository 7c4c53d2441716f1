// Routed experts with 4-bit weights in groups: out[r] = sum over slots of wts * down_e(silu(gate_e x) * (up_e x)).
//
// The rows' picks are sorted by expert and cut into items (an expert and up to 16 Q4_MT of its pairs); a block multiplies
// an item's rows by one tile of the expert's gate|up (8 columns of each) and writes the activated pairs; another multiplies
// those by one tile of the down projection; the last launch adds a row's slots in order. A pair's values depend neither on
// the others of its item nor on their order, so the results are the same on every run.
#include <hip/hip_runtime.h>

#include <type_traits>

#include "ea_host.hpp"
#include "ea_q4.hpp"

namespace ea {

constexpr int Q4_MT = 4;
constexpr uint32_t Q4_MAX_EXPERTS = 4096;

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
    int32_t *sorted, *nitems;
    Q4Item* items;
    uint16_t* h;  // bf16 [terms][pairs][width]
    float* y;     // fp32 [pairs][dims]
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
        const uint32_t e = e0 + t, c = e < a.experts ? count[e] : 0, n = (c + 16 * Q4_MT - 1) / (16 * Q4_MT);
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
            a.items[item + i] = Q4Item{(int32_t)e, (int32_t)(first + i * 16 * Q4_MT),
                                       (int32_t)min(c - i * 16 * Q4_MT, 16u * Q4_MT), 0};
        __syncthreads();
    }
    if (t == 0) *a.nitems = (int32_t)ibase;
    for (uint32_t p = t; p < a.pairs; p += 1024) {
        const uint32_t e = (uint32_t)a.pick[p];
        if (e < a.experts) a.sorted[atomicAdd(&start[e], 1u)] = (int32_t)p;
    }
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

template <bool BF, int GPC, int TERMS, int WK>
__global__ void __launch_bounds__(64 * WK) q4_gateup_kernel(Q4MoeArgs a) {
    __shared__ f4v part[WK][1][Q4_MT][64];
    if ((int)blockIdx.y >= *a.nitems) return;
    const Q4Item it = a.items[blockIdx.y];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t tile = blockIdx.x, chunks = q4_chunks(a.dims);
    const uint8_t* w = a.gu + (size_t)it.expert * a.gu_bytes + (size_t)tile * chunks * q4_chunk_bytes(GPC);
    const uint16_t* row[Q4_MT];
    f4v out[1][Q4_MT];
#pragma unroll
    for (int mt = 0; mt < Q4_MT; ++mt) {
        const int i = min(16 * mt + (lane & 15), it.count - 1);
        row[mt] = a.x + (size_t)((uint32_t)a.sorted[it.first + i] / a.slots) * a.x_stride;
        out[0][mt] = f4v{0.0f, 0.0f, 0.0f, 0.0f};
    }
    q4_stream<BF, GPC, Q4_MT, 1, 1>(w, 0, wave, WK, chunks, row, a.dims, lane, a.sbf, out);
#pragma unroll
    for (int mt = 0; mt < Q4_MT; ++mt) part[wave][0][mt][lane] = out[0][mt];
    __syncthreads();
    for (int i = threadIdx.x; i < 128 * Q4_MT; i += 64 * WK) {
        const int mt = i >> 7, r = (i >> 3) & 15, n = i & 7, at = 16 * mt + r;
        const uint32_t col = tile * 8 + n;
        if (at >= it.count || col >= a.width) continue;
        const float v = swiglu(q4_total<WK, 1, Q4_MT>(part, 0, mt, r, n), q4_total<WK, 1, Q4_MT>(part, 0, mt, r, n + 8));
        store_terms<TERMS>(a.h, (size_t)a.pairs * a.width, (size_t)(it.first + at) * a.width + col, v);
    }
}

template <int GPC, int TERMS, int WK>
__global__ void __launch_bounds__(64 * WK) q4_down_kernel(Q4MoeArgs a) {
    __shared__ f4v part[WK][1][Q4_MT][64];
    if ((int)blockIdx.y >= *a.nitems) return;
    const Q4Item it = a.items[blockIdx.y];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t tile = blockIdx.x, chunks = q4_chunks(a.width);
    const uint8_t* w = a.down + (size_t)it.expert * a.down_bytes + (size_t)tile * chunks * q4_chunk_bytes(GPC);
    f4v out[1][Q4_MT];
#pragma unroll
    for (int mt = 0; mt < Q4_MT; ++mt) out[0][mt] = f4v{0.0f, 0.0f, 0.0f, 0.0f};
    for (uint32_t c = wave; c < chunks; c += WK) {
        const uint8_t* p = w + (size_t)c * q4_chunk_bytes(GPC);
        const u4v words[1] = {reinterpret_cast<const u4v*>(p)[lane]};
        const Q4Params<GPC> par[1] = {q4_params<GPC>(p, lane)};
#pragma unroll
        for (int term = 0; term < TERMS; ++term) {
            u4v x[Q4_MT][4];
#pragma unroll
            for (int mt = 0; mt < Q4_MT; ++mt) {
                const int i = min(16 * mt + (lane & 15), it.count - 1);
                q4_rows(a.h + ((size_t)term * a.pairs + it.first + i) * a.width, c, a.width, lane, x[mt]);
            }
            q4_chunk<true, GPC, Q4_MT, 1>(words, par, x, a.sbf, out);
        }
    }
#pragma unroll
    for (int mt = 0; mt < Q4_MT; ++mt) part[wave][0][mt][lane] = out[0][mt];
    __syncthreads();
    for (int i = threadIdx.x; i < 256 * Q4_MT; i += 64 * WK) {
        const int mt = i >> 8, r = (i >> 4) & 15, n = i & 15, at = 16 * mt + r;
        const uint32_t col = tile * 16 + n;
        if (at >= it.count || col >= a.dims) continue;
        a.y[(size_t)a.sorted[it.first + at] * a.dims + col] = q4_total<WK, 1, Q4_MT>(part, 0, mt, r, n);
    }
}

__global__ void __launch_bounds__(256) q4_combine_kernel(Q4MoeArgs a) {
    const uint32_t r = blockIdx.x, d = blockIdx.y * 256 + threadIdx.x;
    if (d >= a.dims) return;
    float v = 0.0f;
    for (uint32_t k = 0; k < a.slots; ++k) {
        const uint32_t p = r * a.slots + k;
        if ((uint32_t)a.pick[p] < a.experts) v = __builtin_fmaf(a.wts[p], a.y[(size_t)p * a.dims + d], v);
    }
    store_act(a.out, a.out_dtype, (size_t)r * a.dims + d, v);
}

// ---- up to 16 rows --------------------------------------------------------------------------------------------------
// Every distinct expert is multiplied with all rows (an MFMA takes 16 whether they are there or not), so nothing is
// sorted: block (tiles, pair) works if no earlier pair names its expert. h is kept by pair; a row that names an expert twice
// has it twice.
constexpr uint32_t Q4_ROWS = 16, Q4_PAIRS = Q4_ROWS * 32;

template <bool BF, int GPC, int TERMS, int NT, int WK, int NB>
__global__ void __launch_bounds__(64 * WK) q4_gateup_rows_kernel(Q4MoeArgs a) {
    __shared__ f4v part[WK][NT][1][64];
    __shared__ int32_t picks[Q4_PAIRS];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t u = blockIdx.y, chunks = q4_chunks(a.dims), tiles = (a.width + 7) / 8;
    for (uint32_t p = threadIdx.x; p < a.pairs; p += 64 * WK) picks[p] = a.pick[p];
    __syncthreads();
    const int32_t e = picks[u];
    if ((uint32_t)e >= a.experts) return;
    bool before = false;
    for (uint32_t p = lane; p < u; p += 64) before |= picks[p] == e;
    if (__ballot(before)) return;
    const uint32_t first = min(blockIdx.x * NT, tiles - NT);  // the last block's tiles overlap
    const size_t tile_bytes = (size_t)chunks * q4_chunk_bytes(GPC);
    const uint16_t* row[1] = {a.x + (size_t)min((uint32_t)(lane & 15), a.rows - 1) * a.x_stride};
    f4v out[NT][1];
#pragma unroll
    for (int t = 0; t < NT; ++t) out[t][0] = f4v{0.0f, 0.0f, 0.0f, 0.0f};
    q4_stream<BF, GPC, 1, NT, NB>(a.gu + (size_t)e * a.gu_bytes + first * tile_bytes, tile_bytes, wave, WK, chunks, row,
                                  a.dims, lane, a.sbf, out);
#pragma unroll
    for (int t = 0; t < NT; ++t) part[wave][t][0][lane] = out[t][0];
    __syncthreads();
    for (int i = threadIdx.x; i < 128 * NT; i += 64 * WK) {
        const int n = i & 7, t = (i >> 3) % NT, r = i / (8 * NT);
        const uint32_t col = (first + t) * 8 + n;
        if ((uint32_t)r >= a.rows || col >= a.width) continue;
        const float v = swiglu(q4_total<WK, NT, 1>(part, t, 0, r, n), q4_total<WK, NT, 1>(part, t, 0, r, n + 8));
        for (uint32_t k = 0; k < a.slots; ++k) {
            const uint32_t p = r * a.slots + k;
            if (picks[p] == e) store_terms<TERMS>(a.h, (size_t)a.pairs * a.width, (size_t)p * a.width + col, v);
        }
    }
}

// NT tiles of the output for all rows: the waves take the (distinct expert, chunk) units in turn. An activated value's terms
// are rows of their own (term t of row r is row t * rows + r of up to 48), so few rows need one product for all terms; a
// unit's sums are weighted into the wave's fp32 sums, and terms and waves are added at the end.
template <int GPC, int TERMS, int MT, int NT, int WK, int NB>
__global__ void __launch_bounds__(64 * WK) q4_down_rows_kernel(Q4MoeArgs a) {
    __shared__ union {
        f4v part[WK][NT][MT][64];
        struct {
            int32_t expert[Q4_PAIRS];
            float weight[Q4_PAIRS][Q4_ROWS];   // [distinct][row]: the row's weight, 0 where it did not pick the expert
            int16_t pair[Q4_PAIRS][Q4_ROWS];   // its pair, -1
        } d;
    } sh;
    __shared__ int32_t picks[Q4_PAIRS];
    __shared__ uint8_t seen[Q4_PAIRS];
    __shared__ int ndistinct;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    static_assert(64 * WK >= Q4_PAIRS, "a thread a pair");
    for (uint32_t p = threadIdx.x; p < a.pairs; p += 64 * WK) {
        picks[p] = a.pick[p];
        seen[p] = 0;
    }
    __syncthreads();
    {  // whether an earlier pair names the same expert: as many threads a pair as there are
        const uint32_t per = 64 * WK / a.pairs, p = threadIdx.x / per, sub = threadIdx.x % per;
        if (p < a.pairs) {
            const int32_t e = picks[p];
            bool again = (uint32_t)e >= a.experts;
#pragma unroll 4
            for (uint32_t q = sub; q < p; q += per) again |= picks[q] == e;
            if (again) seen[p] = 1;
        }
    }
    __syncthreads();
    if (wave == 0) {  // the distinct experts in the order of their first pairs
        int n = 0;
        for (uint32_t p0 = 0; p0 < a.pairs; p0 += 64) {
            const bool fresh = p0 + lane < a.pairs && !seen[p0 + lane];
            const uint64_t all = __ballot(fresh);
            if (fresh) sh.d.expert[n + __builtin_popcountll(all & ((1ull << lane) - 1))] = picks[p0 + lane];
            n += __builtin_popcountll(all);
        }
        if (lane == 0) ndistinct = n;
    }
    __syncthreads();
    const int nd = ndistinct;
    for (int i = threadIdx.x; i < nd * (int)Q4_ROWS; i += 64 * WK) {
        const int d = i / (int)Q4_ROWS, r = i % (int)Q4_ROWS;
        const int32_t e = sh.d.expert[d];
        float w = 0.0f;
        int at = -1;
        if ((uint32_t)r < a.rows)
            for (uint32_t k = 0; k < a.slots; ++k)
                if (picks[r * a.slots + k] == e) {
                    w = w + a.wts[r * a.slots + k];
                    at = (int)(r * a.slots + k);
                }
        sh.d.weight[d][r] = w;
        sh.d.pair[d][r] = (int16_t)at;
    }
    __syncthreads();
    const uint32_t chunks = q4_chunks(a.width), tiles = q4_tiles(a.dims), first = min(blockIdx.x * NT, tiles - NT);
    const size_t tile_bytes = (size_t)chunks * q4_chunk_bytes(GPC), plane = (size_t)a.pairs * a.width;
    const uint8_t* w0 = a.down + first * tile_bytes;
    f4v out[NT][MT];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) out[t][mt] = f4v{0.0f, 0.0f, 0.0f, 0.0f};
    // the lane's rows: as A operand, row 16 mt + (lane & 15); in the sums, rows 16 mt + 4 (lane >> 4) + i
    const uint32_t units = nd * chunks;
    for (uint32_t u0 = wave; u0 < units; u0 += WK * NB) {
        u4v words[NB][NT], x[NB][MT][4];
        Q4Params<GPC> par[NB][NT];
#pragma unroll
        for (int i = 0; i < NB; ++i) {
            const uint32_t u = min(u0 + WK * i, units - 1), d = u / chunks, c = u - d * chunks;
            const uint8_t* p = w0 + (size_t)sh.d.expert[d] * a.down_bytes + (size_t)c * q4_chunk_bytes(GPC);
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                words[i][t] = reinterpret_cast<const u4v*>(p + t * tile_bytes)[lane];
                par[i][t] = q4_params<GPC>(p + t * tile_bytes, lane);
            }
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
                const uint32_t v = 16 * mt + (lane & 15), term = v / a.rows;
                const int at = term < TERMS ? sh.d.pair[d][v - term * a.rows] : -1;
#pragma unroll
                for (int j = 0; j < 4; ++j) x[i][mt][j] = u4v{0, 0, 0, 0};
                if (at >= 0) q4_rows(a.h + term * plane + (size_t)at * a.width, c, a.width, lane, x[i][mt]);
            }
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < NB; ++i) {
            if (u0 + WK * i >= units) break;
            const uint32_t d = (u0 + WK * i) / chunks;
            f4v y[NT][MT];
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) y[t][mt] = f4v{0.0f, 0.0f, 0.0f, 0.0f};
            q4_chunk<true, GPC, MT, NT>(words[i], par[i], x[i], a.sbf, y);
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const uint32_t v = 16 * mt + 4 * (lane >> 4) + r, term = v / a.rows;
                    const float wt = term < TERMS ? sh.d.weight[d][v - term * a.rows] : 0.0f;
#pragma unroll
                    for (int t = 0; t < NT; ++t) out[t][mt][r] = __builtin_fmaf(wt, y[t][mt][r], out[t][mt][r]);
                }
        }
    }
    __syncthreads();  // the tables are done with
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) sh.part[wave][t][mt][lane] = out[t][mt];
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < 16 * NT * a.rows; i += 64 * WK) {
        const int n = i & 15, t = (i >> 4) % NT;
        const uint32_t r = i / (16 * NT), col = (first + t) * 16 + n;
        if (col >= a.dims) continue;
        float v = 0.0f;
#pragma unroll
        for (int k = TERMS - 1; k >= 0; --k) {  // the small terms first
            const uint32_t vr = k * a.rows + r;
            v = v + q4_total<WK, NT, MT>(sh.part, t, vr >> 4, vr & 15, n);
        }
        store_act(a.out, a.out_dtype, (size_t)r * a.dims + col, v);
    }
}

template <int GPC, int TERMS>
static void launch_rows(hipStream_t s, const Q4MoeArgs& a, bool bf) {
    const unsigned tiles = (a.width + 7) / 8, dtiles = q4_tiles(a.dims);
    auto gateup = [&](auto bf_) {
        constexpr bool BF = decltype(bf_)::value;
        if (a.rows <= 4 || tiles < 2) q4_gateup_rows_kernel<BF, GPC, TERMS, 1, 8, 3><<<dim3(tiles, a.pairs), 512, 0, s>>>(a);
        else q4_gateup_rows_kernel<BF, GPC, TERMS, 2, 8, 3><<<dim3((tiles + 1) / 2, a.pairs), 512, 0, s>>>(a);
    };
    if (bf) gateup(std::true_type{});
    else gateup(std::false_type{});
    auto down = [&](auto mt_) {
        constexpr int MT = decltype(mt_)::value;
        q4_down_rows_kernel<GPC, TERMS, MT, 1, 8, 2><<<dtiles, 512, 0, s>>>(a);
    };
    const uint32_t groups = (a.rows * TERMS + 15) / 16;
    if (groups == 1) down(std::integral_constant<int, 1>{});
    else if (TERMS > 1 && groups == 2) down(std::integral_constant<int, TERMS < 2 ? 1 : 2>{});
    else down(std::integral_constant<int, TERMS>{});
}

template <int GPC, int TERMS>
static void launch_items(hipStream_t s, const Q4MoeArgs& a, bool bf, uint32_t max_items) {
    const dim3 gu((a.width + 7) / 8, max_items), dn((a.dims + 15) / 16, max_items);
    if (bf) q4_gateup_kernel<true, GPC, TERMS, 4><<<gu, 256, 0, s>>>(a);
    else q4_gateup_kernel<false, GPC, TERMS, 4><<<gu, 256, 0, s>>>(a);
    q4_down_kernel<GPC, TERMS, 2><<<dn, 128, 0, s>>>(a);
}

// Terms of the activated values: what the output's type can show (bf16 8 bits, fp16 11, fp32 24).
static int q4_terms(int out_dtype) { return out_dtype == BF16 ? 1 : out_dtype == F16 ? 2 : 3; }

static uint32_t q4_max_items(uint32_t experts, size_t pairs) {
    const size_t full = pairs / (16 * Q4_MT), some = pairs < experts ? pairs : experts;
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
    if (q4_experts_ok(ex) || rows == 0 || rows > EA_Q4_MAX_ROWS || slots == 0 || slots > 32) return 0;
    return q4_carve(&s, 0, ex, rows, slots);
}

int ea_q4_scratch_init(ea_q4_scratch* s, void* base, size_t bytes, const ea_q4_experts* ex, uint32_t rows,
                       uint32_t slots) {
    int r = q4_experts_ok(ex);
    if (r) return r;
    if (!s || !base || (reinterpret_cast<uintptr_t>(base) & 255) || rows == 0 || rows > EA_Q4_MAX_ROWS) return EA_BAD_ARGUMENT;
    if (slots == 0 || slots > 32) return EA_TOO_MANY_SLOTS;
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
    if (R <= Q4_ROWS) {
        auto go = [&](auto gpc_) {
            constexpr int GPC = decltype(gpc_)::value;
            if (terms == 1) launch_rows<GPC, 1>(s, a, x_dtype == BF16);
            else if (terms == 2) launch_rows<GPC, 2>(s, a, x_dtype == BF16);
            else launch_rows<GPC, 3>(s, a, x_dtype == BF16);
        };
        if (gpc == 4) go(std::integral_constant<int, 4>{});
        else if (gpc == 2) go(std::integral_constant<int, 2>{});
        else go(std::integral_constant<int, 1>{});
        return launched();
    }
    q4_group_kernel<<<1, 1024, 0, s>>>(a);
    auto go = [&](auto gpc_) {
        constexpr int GPC = decltype(gpc_)::value;
        if (terms == 1) launch_items<GPC, 1>(s, a, x_dtype == BF16, max_items);
        else if (terms == 2) launch_items<GPC, 2>(s, a, x_dtype == BF16, max_items);
        else launch_items<GPC, 3>(s, a, x_dtype == BF16, max_items);
    };
    if (gpc == 4) go(std::integral_constant<int, 4>{});
    else if (gpc == 2) go(std::integral_constant<int, 2>{});
    else go(std::integral_constant<int, 1>{});
    q4_combine_kernel<<<dim3(R, (a.dims + 255) / 256), 256, 0, s>>>(a);
    return launched();
}

}  // extern "C"
