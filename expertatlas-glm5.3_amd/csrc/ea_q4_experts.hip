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

// The waves' sums of one tile in wave order, for row r and weight row n.
template <int MT, int WK>
__device__ __forceinline__ float q4_total(const f4v (&part)[WK][MT][64], int mt, int r, int n) {
    const float* all = reinterpret_cast<const float*>(part);
    const int slot = (mt * 64 + (r >> 2) * 16 + n) * 4 + (r & 3);
    float v = all[slot];
#pragma unroll
    for (int k = 1; k < WK; ++k) v = v + all[k * MT * 256 + slot];
    return v;
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
    __shared__ f4v part[WK][Q4_MT][64];
    if ((int)blockIdx.y >= *a.nitems) return;
    const Q4Item it = a.items[blockIdx.y];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint32_t tile = blockIdx.x, chunks = q4_chunks(a.dims);
    const uint8_t* w = a.gu + (size_t)it.expert * a.gu_bytes + (size_t)tile * chunks * q4_chunk_bytes(GPC);
    const uint16_t* row[Q4_MT];
    f4v out[Q4_MT];
#pragma unroll
    for (int mt = 0; mt < Q4_MT; ++mt) {
        const int i = min(16 * mt + (lane & 15), it.count - 1);
        row[mt] = a.x + (size_t)((uint32_t)a.sorted[it.first + i] / a.slots) * a.x_stride;
        out[mt] = f4v{0.0f, 0.0f, 0.0f, 0.0f};
    }
    for (uint32_t c = wave; c < chunks; c += WK) {
        const uint8_t* p = w + (size_t)c * q4_chunk_bytes(GPC);
        const u4v words = reinterpret_cast<const u4v*>(p)[lane];
        const auto par = q4_params<GPC>(p, lane);
        u4v x[Q4_MT][4];
#pragma unroll
        for (int mt = 0; mt < Q4_MT; ++mt) q4_rows(row[mt], c, a.dims, lane, x[mt]);
        q4_chunk<BF, GPC, Q4_MT>(words, par, x, a.sbf, out);
    }
#pragma unroll
    for (int mt = 0; mt < Q4_MT; ++mt) part[wave][mt][lane] = out[mt];
    __syncthreads();
    for (int i = threadIdx.x; i < 128 * Q4_MT; i += 64 * WK) {
        const int mt = i >> 7, r = (i >> 3) & 15, n = i & 7, at = 16 * mt + r;
        const uint32_t col = tile * 8 + n;
        if (at >= it.count || col >= a.width) continue;
        const float v = swiglu(q4_total<Q4_MT, WK>(part, mt, r, n), q4_total<Q4_MT, WK>(part, mt, r, n + 8));
        store_terms<TERMS>(a.h, (size_t)a.pairs * a.width, (size_t)(it.first + at) * a.width + col, v);
    }
}

template <int GPC, int TERMS, int WK>
__global__ void __launch_bounds__(64 * WK) q4_down_kernel(Q4MoeArgs a) {
    __shared__ f4v part[WK][Q4_MT][64];
    if ((int)blockIdx.y >= *a.nitems) return;
    const Q4Item it = a.items[blockIdx.y];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint32_t tile = blockIdx.x, chunks = q4_chunks(a.width);
    const uint8_t* w = a.down + (size_t)it.expert * a.down_bytes + (size_t)tile * chunks * q4_chunk_bytes(GPC);
    f4v out[Q4_MT];
#pragma unroll
    for (int mt = 0; mt < Q4_MT; ++mt) out[mt] = f4v{0.0f, 0.0f, 0.0f, 0.0f};
    for (uint32_t c = wave; c < chunks; c += WK) {
        const uint8_t* p = w + (size_t)c * q4_chunk_bytes(GPC);
        const u4v words = reinterpret_cast<const u4v*>(p)[lane];
        const auto par = q4_params<GPC>(p, lane);
#pragma unroll
        for (int term = 0; term < TERMS; ++term) {
            u4v x[Q4_MT][4];
#pragma unroll
            for (int mt = 0; mt < Q4_MT; ++mt) {
                const int i = min(16 * mt + (lane & 15), it.count - 1);
                q4_rows(a.h + ((size_t)term * a.pairs + it.first + i) * a.width, c, a.width, lane, x[mt]);
            }
            q4_chunk<true, GPC, Q4_MT>(words, par, x, a.sbf, out);
        }
    }
#pragma unroll
    for (int mt = 0; mt < Q4_MT; ++mt) part[wave][mt][lane] = out[mt];
    __syncthreads();
    for (int i = threadIdx.x; i < 256 * Q4_MT; i += 64 * WK) {
        const int mt = i >> 8, r = (i >> 4) & 15, n = i & 15, at = 16 * mt + r;
        const uint32_t col = tile * 16 + n;
        if (at >= it.count || col >= a.dims) continue;
        a.y[(size_t)a.sorted[it.first + at] * a.dims + col] = q4_total<Q4_MT, WK>(part, mt, r, n);
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
