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

// Few rows: a block takes NT tiles of one job and up to 16 rows; its WK waves take every WK-th chunk and add their sums in wave
// order. Bound by the weights' bandwidth where there are many, by latencies where there are few; from then on by the rows,
// which every block reads from L2, so wide jobs take four tiles a block, which share them: 65521 x 6144 at 1 / 8 / 16 rows
// 41 / 46 / 54 us with four tiles (226 MB: 5.5 TB/s), 44 / 55 / 74 with two, 57 / 86 / 118 with one; 8192 x 6144 at one row
// 11.3, 8.4 and 9.6 us, 4096 x 6144 9.8, 6.7 and 5.6, where more tiles a block leave the card idle. 2048 x 6144: 5.4 us.
// More than 16 rows are cut into groups of 16 where all blocks then run at once and a row is long: 32 rows x 2048 x 6144 take
// 9.0 us so, 14.4 in blocks of 32 rows; but 48 rows 15.0 and 14.6, and 64 x 512 x 2048 8.1 and 7.3.
template <bool BF, bool SBF, int GPC, int NT, int WK, int NB>
__global__ void __launch_bounds__(64 * WK) q4_linear_kernel(Q4LinArgs a) {
    __shared__ f4v part[WK][NT][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const Q4Job job = a.job[blockIdx.z];
    const uint32_t tiles = q4_tiles(job.n), tile0 = blockIdx.x * NT;
    if (tile0 >= tiles) return;
    const size_t tile_bytes = (size_t)a.chunks * q4_chunk_bytes(GPC);
    const uint32_t own = min(tiles, (uint32_t)NT), first = min(tile0, tiles - own);  // the last block's tiles overlap
    const uint32_t m0 = blockIdx.y * 16, m = min(a.m - m0, 16u);
    const uint16_t* row = a.x + (size_t)(m0 + min((uint32_t)(lane & 15), m - 1)) * a.x_stride;  // past m the last row again
    f4v out[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) out[t] = f4v{0.0f, 0.0f, 0.0f, 0.0f};
    q4_stream<BF, SBF, GPC, NT, NB>(job.w + first * tile_bytes, tile_bytes, wave, WK, a.chunks, row, a.k, lane, out, own - 1);
#pragma unroll
    for (int t = 0; t < NT; ++t) part[wave][t][lane] = out[t];
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < 16 * NT * m; i += 64 * WK) {
        const uint32_t n = i & 15, t = (i >> 4) % NT, r = i / (16 * NT), col = (first + t) * 16 + n;
        if (col < job.n) store_act(job.y, job.y_dtype, (size_t)(m0 + r) * job.n + col, q4_total<WK, NT>(part, t, r, n));
    }
}

// More rows: a block takes 16 MT rows and 4 NT tiles, and KS groups of four waves every KS-th chunk of them: each group stages
// its chunk's rows in LDS, in two buffers, while the chunk before is multiplied, and reads its weights a chunk ahead; the
// groups' sums are added in order at the end. Four groups of one tile a wave where that makes at most 256 blocks, else two of
// two tiles: 128 rows x 2048 x 6144 15.5 against 24.8 us, 64 x 8192 x 2048 8.7 against 11.8, but 128 x 6144 x 2048 13.7
// against 12.5, 301 x 6144 x 2048 26.5 against 18 (420 TFLOP/s). Bound by the instructions beside the products of rows and
// weights: the rows' sums are products against ones in every wave, a third of its matrix instructions with two tiles and
// half with one, and conversions, scales and biases take the vector units. Waves count more than large tiles: 512 rows x
// 12000 x 8192 took 189 us with 32 rows, two tiles and two groups, 198 with 64 rows, 212 without groups (196 to 240 us for the
// first of these from one run to the next).
template <bool BF, bool SBF, int GPC, int MT, int NT, int KS>
__global__ void __launch_bounds__(256 * KS) q4_linear_split_kernel(Q4LinArgs a) {
    constexpr int BUFFER = MT * 4096, PARTS = KS * 4 * NT * MT * 1024;
    __shared__ __attribute__((aligned(16))) uint8_t lds[2 * KS * BUFFER > PARTS ? 2 * KS * BUFFER : PARTS];
    const Q4Job job = a.job[blockIdx.z];
    const uint32_t tiles = q4_tiles(job.n), m0 = blockIdx.y * 16 * MT;
    if (blockIdx.x * 4 * NT >= tiles) return;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6 & 3);
    const uint32_t group = __builtin_amdgcn_readfirstlane(threadIdx.x >> 8), t256 = threadIdx.x & 255;
    const uint32_t piece = t256 & 15, row0 = t256 >> 4, to = row0 * 256 + 16 * (piece ^ row0);
    uint8_t* const mine = lds + group * 2 * BUFFER;
    const uint8_t* w[NT];
    const uint16_t* src[MT];
#pragma unroll
    for (int t = 0; t < NT; ++t)
        w[t] = job.w + (size_t)min((blockIdx.x * 4 + wave) * NT + t, tiles - 1) * a.chunks * q4_chunk_bytes(GPC);
#pragma unroll
    for (int i = 0; i < MT; ++i) src[i] = a.x + (size_t)min(m0 + row0 + 16 * i, a.m - 1) * a.x_stride;
    u4v ra[MT], rw[2][NT];
    Q4Params<GPC> rp[2][NT];
    const auto load = [&](int set, uint32_t c) {
        c = min(c, a.chunks - 1);
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const uint8_t* p = w[t] + (size_t)c * q4_chunk_bytes(GPC);
            rw[set][t] = reinterpret_cast<const u4v*>(p)[lane];
            rp[set][t] = q4_params<GPC>(p, lane);
        }
        const uint32_t at = c * Q4_CHUNK + 8 * piece, off = at < a.k ? at : a.k - 32 + 8 * (piece & 3);
#pragma unroll
        for (int i = 0; i < MT; ++i) ra[i] = *reinterpret_cast<const u4v_a8*>(src[i] + off);
    };
    f4v out[NT][MT];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) out[t][mt] = f4v{0.0f, 0.0f, 0.0f, 0.0f};
    const auto step = [&](auto set_, uint32_t c) __attribute__((always_inline)) {  // every group takes every step
        constexpr int SET = decltype(set_)::value;
#pragma unroll
        for (int i = 0; i < MT; ++i) *reinterpret_cast<u4v*>(mine + SET * BUFFER + to + 4096 * i) = ra[i];
        load(1 - SET, c + KS);
        __syncthreads();
        if (c < a.chunks) q4_gemm_chunk<BF, SBF, GPC, MT, NT, true>(mine + SET * BUFFER, rw[SET], rp[SET], lane, out);
    };
    load(0, group);
    for (uint32_t c0 = 0; c0 < a.chunks; c0 += 2 * KS) {
        step(std::integral_constant<int, 0>{}, c0 + group);
        if (c0 + KS < a.chunks) step(std::integral_constant<int, 1>{}, c0 + KS + group);
    }
    __syncthreads();
    f4v(*part)[4][NT][MT][64] = reinterpret_cast<f4v(*)[4][NT][MT][64]>(lds);
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) part[group][wave][t][mt][lane] = out[t][mt];
    __syncthreads();
    for (int i = threadIdx.x; i < 4 * NT * MT * 256; i += 256 * KS) {
        const int n = i & 15, t = (i >> 4) % (4 * NT), r = (i / (64 * NT)) & 15, mt = i / (1024 * NT);
        const uint32_t mr = m0 + 16 * mt + r, nc = (blockIdx.x * 4 * NT + t) * 16 + n;
        if (mr >= a.m || nc >= job.n) continue;
        const float* p = reinterpret_cast<const float*>(lds) + ((t * MT + mt) * 64 + (r >> 2) * 16 + n) * 4 + (r & 3);
        float v = p[0];
#pragma unroll
        for (int g = 1; g < KS; ++g) v = v + p[g * 4 * NT * MT * 256];
        store_act(job.y, job.y_dtype, (size_t)mr * job.n + nc, v);
    }
}

static int launch_linear(hipStream_t s, const Q4LinArgs& a, uint32_t tiles, bool bf, bool sbf, int gpc) {
    auto go = [&](auto gpc_, auto bf_, auto sbf_) {
        constexpr int GPC = decltype(gpc_)::value;
        constexpr bool BF = decltype(bf_)::value, SBF = decltype(sbf_)::value;
        const unsigned jobs = (unsigned)a.jobs;
        const unsigned groups = (a.m + 15) / 16;
        const auto blocks = [&](uint32_t nt, uint32_t rows) {
            return dim3((tiles + nt - 1) / nt, (a.m + rows - 1) / rows, jobs);
        };
        if (groups == 1 || ((uint64_t)tiles * jobs * groups <= 256 && a.chunks > 16)) {
            if (tiles * jobs < 512) q4_linear_kernel<BF, SBF, GPC, 1, 16, 3><<<blocks(1, 16), 1024, 0, s>>>(a);
            else if (tiles * jobs < 1536) q4_linear_kernel<BF, SBF, GPC, 2, 8, 3><<<blocks(2, 16), 512, 0, s>>>(a);
            else q4_linear_kernel<BF, SBF, GPC, 4, 8, 2><<<blocks(4, 16), 512, 0, s>>>(a);
            return;
        }
        const dim3 one = blocks(4, 32);  // four waves of a tile each
        if ((uint64_t)one.x * one.y * jobs <= 256) q4_linear_split_kernel<BF, SBF, GPC, 2, 1, 4><<<one, 1024, 0, s>>>(a);
        else q4_linear_split_kernel<BF, SBF, GPC, 2, 2, 2><<<blocks(8, 32), 512, 0, s>>>(a);
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
        if (!l || !l->words || (l->words & 15) || !outs[j]) return EA_BAD_ARGUMENT;
        if (out_dtypes[j] < F16 || out_dtypes[j] > F32) return EA_BAD_ARGUMENT;
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
