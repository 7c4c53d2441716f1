// 4-bit affine weights: the layout's packing and the linears (ea_q4.hpp has the format and the products).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "ea_host.hpp"
#include "ea_q4_gemm.hpp"

namespace ea {

// ---- packing ----------------------------------------------------------------------------------------------------
// A wave a (tile, chunk): its lanes fetch the source words of their row and spread each one's eight values over the
// half-bytes. With two sources (gate and up of experts) a tile holds 8 rows of each, so that one block has both factors of a
// column of the SwiGLU.
struct PackSrc {
    const uint32_t* words;
    const uint16_t *s, *b;
};

__global__ void __launch_bounds__(256) q4_pack_kernel(PackSrc s0, PackSrc s1, uint8_t* __restrict__ out, uint32_t n,
                                                      uint32_t k, int gpc, bool bf, uint32_t tiles, uint32_t chunks,
                                                      size_t units) {
    const size_t unit = (size_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (unit >= units) return;
    const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
    const uint32_t c = (uint32_t)(unit % chunks);
    const size_t mt = unit / chunks, m = mt / tiles;
    const uint32_t t = (uint32_t)(mt % tiles);
    const bool two = s1.words != nullptr;
    const PackSrc src = two && r >= 8 ? s1 : s0;
    const uint32_t row = two ? t * 8 + (r & 7) : t * 16 + r;
    uint8_t* to = out + unit * q4_chunk_bytes(gpc);
    const size_t at = m * n + row;  // the row among all matrices' rows
    u4v v;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const uint32_t k0 = c * Q4_CHUNK + 32 * j + 8 * g;
        const uint32_t w = row < n && k0 < k ? src.words[at * (k / 8) + k0 / 8] : 0u;
        uint32_t o = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) o |= (w >> (4 * i) & 15u) << (i < 4 ? 8 * i : 8 * (i - 4) + 4);
        v[j] = o;
    }
    reinterpret_cast<u4v*>(to)[lane] = v;
    const uint32_t group = Q4_CHUNK / gpc;
    for (int q = g; q < gpc; q += 4) {
        const uint32_t gi = (c * Q4_CHUNK) / group + q;
        uint32_t p = 0;
        if (row < n && gi < k / group) {
            const size_t i = at * (k / group) + gi;
            const uint16_t s = src.s[i];
            // without biases the integers stand for q - 8: b = -8 s, exact in bf16 and, up to 8191, in fp16
            const uint16_t b = src.b ? src.b[i] : bf ? f2bf(-8.0f * bf2f(s)) : f2h(-8.0f * h2f(s));
            p = (uint32_t)s | (uint32_t)b << 16;
        }
        reinterpret_cast<uint32_t*>(to + Q4_WORDS)[r * gpc + q] = p;
    }
}

// ---- linears ----------------------------------------------------------------------------------------------------
struct Q4Job {
    const uint8_t* w;
    void* y;
    uint32_t n;
    int y_dtype;
};
struct Q4LinArgs {
    Q4Job job[EA_MAX_JOBS];
    const uint16_t* x;
    size_t x_stride;
    uint32_t m, k, chunks;
    int jobs;
};

// A block takes NT tiles of one job and 16 MT rows; its WK waves take every WK-th chunk and add their sums in wave order.
template <bool BF, bool SBF, int GPC, int MT, int NT, int WK, int NB>
__global__ void __launch_bounds__(64 * WK) q4_linear_kernel(Q4LinArgs a) {
    __shared__ f4v part[WK][NT][MT][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const Q4Job job = a.job[blockIdx.z];
    const uint32_t tiles = q4_tiles(job.n), tile0 = blockIdx.x * NT, m0 = blockIdx.y * 16 * MT;
    if (tile0 >= tiles) return;
    const size_t tile_bytes = (size_t)a.chunks * q4_chunk_bytes(GPC);
    const uint32_t first = NT > 1 ? min(tile0, tiles - min(tiles, (uint32_t)NT)) : tile0;  // the last block's tiles overlap
    const uint16_t* row[MT];
    f4v out[NT][MT];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
        row[mt] = a.x + (size_t)min(m0 + 16 * mt + (lane & 15), a.m - 1) * a.x_stride;  // rows past m re-read the last
#pragma unroll
        for (int t = 0; t < NT; ++t) out[t][mt] = f4v{0.0f, 0.0f, 0.0f, 0.0f};
    }
    q4_stream<BF, SBF, GPC, MT, NT, NB>(job.w + first * tile_bytes, tiles < NT ? 0 : tile_bytes, wave, WK, a.chunks, row, a.k, lane,
                                   out);
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) part[wave][t][mt][lane] = out[t][mt];
    __syncthreads();
    for (int i = threadIdx.x; i < 256 * MT * NT; i += 64 * WK) {
        const int n = i & 15, t = (i >> 4) % NT, r = (i / (16 * NT)) & 15, mt = i / (256 * NT);
        const uint32_t mr = m0 + 16 * mt + r, nc = (first + t) * 16 + n;
        if (mr < a.m && nc < job.n && (NT == 1 || first + t < tiles))
            store_act(job.y, job.y_dtype, (size_t)mr * job.n + nc, q4_total<WK, NT, MT>(part, t, mt, r, n));
    }
}

#ifndef LV
#define LV 2
#endif
#ifndef LAH
#define LAH 1
#endif
// More rows: 16 MT rows and 4 NT tiles a block.
template <bool BF, bool SBF, int GPC, int MT, int NT>
__global__ void __launch_bounds__(Q4_GEMM_THREADS, 2) q4_linear_gemm_kernel(Q4LinArgs a) {
    __shared__ __attribute__((aligned(16))) uint8_t lds[q4_gemm_lds<MT, NT>()];
    const Q4Job job = a.job[blockIdx.z];
    const uint32_t tiles = q4_tiles(job.n), m0 = blockIdx.y * 16 * MT;
    if (blockIdx.x * 4 * NT >= tiles) return;
    const int lane = threadIdx.x & 63;
    q4_gemm<BF, SBF, GPC, MT, NT, true, false, LAH>(
        lds, job.w, tiles, a.k, 1, 0, blockIdx.x, 1u << 24,
        [&](uint32_t i) { return a.x + (size_t)min(m0 + i, a.m - 1) * a.x_stride; }, nullptr,
        [&](uint32_t r, uint32_t n, const f4v& v) {
            if (m0 + r >= a.m) return;
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (n + i < job.n) store_act(job.y, job.y_dtype, (size_t)(m0 + r) * job.n + n + i, v[i]);
        });
}

static int launch_linear(hipStream_t s, const Q4LinArgs& a, uint32_t tiles, bool bf, bool sbf, int gpc) {
    auto go = [&](auto gpc_, auto bf_, auto sbf_) {
        constexpr int GPC = decltype(gpc_)::value;
        constexpr bool BF = decltype(bf_)::value, SBF = decltype(sbf_)::value;
        const unsigned jobs = (unsigned)a.jobs;
        if (a.m <= 16) {
            if (tiles * jobs < 512) q4_linear_kernel<BF, SBF, GPC, 1, 1, 16, 3><<<dim3(tiles, 1, jobs), 1024, 0, s>>>(a);
            else q4_linear_kernel<BF, SBF, GPC, 1, 2, 8, 3><<<dim3((tiles + 1) / 2, 1, jobs), 512, 0, s>>>(a);
        } else {

            if (LV == 0) q4_linear_kernel<BF, SBF, GPC, 4, 1, 8, 1><<<dim3(tiles, (a.m + 63) / 64, jobs), 512, 0, s>>>(a);
            else q4_linear_gemm_kernel<BF, SBF, GPC, 4, LV ? LV : 1><<<dim3((tiles + 4 * LV - 1) / (4 * (LV ? LV : 1)), (a.m + 63) / 64, jobs), Q4_GEMM_THREADS, 0, s>>>(a);
        }
    };
    q4_types(bf, sbf, gpc, go);
    return launched();
}

static bool q4_group_ok(uint32_t group) { return group == 32 || group == 64 || group == 128; }

}  // namespace ea

using namespace ea;

extern "C" {

size_t ea_q4_bytes(uint32_t n, uint32_t k, uint32_t group) {
    if (!q4_group_ok(group) || n == 0 || k == 0 || k % group != 0) return 0;
    return (size_t)q4_tiles(n) * q4_chunks(k) * q4_chunk_bytes(128 / (int)group);
}

int ea_q4_pack(ea_stream_t stream, const void* words0, const void* scales0, const void* biases0, const void* words1,
               const void* scales1, const void* biases1, void* out, uint32_t n, uint32_t k, uint32_t group, int s_dtype,
               uint32_t count) {
    if (!words0 || !scales0 || !out || (s_dtype != F16 && s_dtype != BF16)) return EA_BAD_ARGUMENT;
    if (!words1 != !scales1 || (words1 && !biases0 != !biases1)) return EA_BAD_ARGUMENT;
    if (!q4_group_ok(group)) return EA_BAD_WIDTH;
    if (n == 0 || k == 0) return EA_BAD_ARGUMENT;
    if (k % group != 0) return EA_UNEVEN_SPLIT;
    if (reinterpret_cast<uintptr_t>(out) & 15) return EA_BAD_ARGUMENT;
    EA_REQUIRE_CTX(ctx_);
    (void)ctx_;
    if (count == 0) return EA_OK;
    const uint32_t tiles = words1 ? n / 8 + (n % 8 != 0) : q4_tiles(n), chunks = q4_chunks(k);
    const size_t units = (size_t)tiles * chunks * count, blocks = (units + 3) / 4;
    if (blocks > 0x7fffffffu) return EA_BAD_ARGUMENT;
    const PackSrc a{static_cast<const uint32_t*>(words0), static_cast<const uint16_t*>(scales0),
                    static_cast<const uint16_t*>(biases0)};
    const PackSrc b{static_cast<const uint32_t*>(words1), static_cast<const uint16_t*>(scales1),
                    static_cast<const uint16_t*>(biases1)};
    q4_pack_kernel<<<(unsigned)blocks, 256, 0, as_stream(stream)>>>(a, b, static_cast<uint8_t*>(out), n, k, 128 / (int)group,
                                                                   s_dtype == BF16, tiles, chunks, units);
    return launched();
}

int ea_q4_call(ea_stream_t stream, const ea_q4_linear* const* ls, uint32_t nls, const void* x, int x_dtype,
               uint32_t x_stride, uint32_t m, const uint64_t* outs, const int* out_dtypes) {
    if (!ls || !outs || !out_dtypes) return EA_BAD_ARGUMENT;
    if (nls == 0 || nls > EA_MAX_JOBS) return EA_NOT_GROUPABLE;
    Q4LinArgs a{};
    uint32_t tiles = 0;
    for (uint32_t j = 0; j < nls; ++j) {
        const ea_q4_linear* l = ls[j];
        if (!l || !l->words || !outs[j] || out_dtypes[j] < F16 || out_dtypes[j] > F32) return EA_BAD_ARGUMENT;
        if (!q4_group_ok(l->group)) return EA_BAD_WIDTH;
        if (l->n == 0 || l->k == 0 || (l->s_dtype != F16 && l->s_dtype != BF16)) return EA_BAD_ARGUMENT;
        if (l->k % l->group != 0) return EA_UNEVEN_SPLIT;
        if (l->k != ls[0]->k || l->group != ls[0]->group || l->s_dtype != ls[0]->s_dtype) return EA_NOT_GROUPABLE;
        a.job[j] = Q4Job{dptr<const uint8_t>(l->words), dptr<void>(outs[j]), l->n, out_dtypes[j]};
        tiles = std::max(tiles, q4_tiles(l->n));
    }
    if (!x || (x_dtype != F16 && x_dtype != BF16) || (reinterpret_cast<uintptr_t>(x) & 7)) return EA_BAD_ARGUMENT;
    if (x_stride < ls[0]->k || x_stride % 4 != 0) return EA_BAD_ROW_STRIDE;
    if (m > EA_Q4_MAX_ROWS) return EA_BAD_ARGUMENT;
    EA_REQUIRE_CTX(ctx_);
    (void)ctx_;
    if (m == 0) return EA_OK;
    a.x = static_cast<const uint16_t*>(x);
    a.x_stride = x_stride;
    a.m = m;
    a.k = ls[0]->k;
    a.chunks = q4_chunks(a.k);
    a.jobs = (int)nls;
    return launch_linear(as_stream(stream), a, tiles, x_dtype == BF16, ls[0]->s_dtype == BF16, 128 / (int)ls[0]->group);
}

}  // extern "C"
