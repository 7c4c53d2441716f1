// Routing to experts in its general form: softmax or sigmoid scores, a bias for balance that takes part in the choice alone,
// groups of experts of which the best are kept, the k largest choices, weights that are renormalised and scaled.
//
// A choice is compared in 64 bits: the picks are whole numbers, two choices can lie closer than a 32-bit sigmoid's error, and
// a balance bias moves them to within it on purpose, so that the picks would otherwise depend on how a sigmoid rounds.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "ea_device.hpp"
#include "ea_host.hpp"

namespace ea {

struct RouteArgs {
    const void* logits;
    const float* bias;
    int32_t* pick;
    float* wts;
    size_t stride;
    uint32_t rows;
    int experts, slots, groups, top_groups, group_best, dtype;
    bool softmax, renorm;
    float scale;
};

// The ranking key of a choice: order_key() in 64 bits. Order-preserving over numbers, NaN 1, and 0 for an expert that is out.
__device__ __forceinline__ uint64_t choice_key(double c) {
    const uint64_t b = __builtin_bit_cast(uint64_t, c + 0.0);
    const uint64_t k = (b >> 63) ? ~b : (b | (1ull << 63));
    return c != c ? 1ull : k;
}
__device__ __forceinline__ double choice_of(uint64_t k) {
    return __builtin_bit_cast(double, (k >> 63) ? k & ~(1ull << 63) : k == 1 ? 0x7ff8000000000000ull : ~k);
}

template <int CTL>
__device__ __forceinline__ uint32_t dpp(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_mov_dpp((int)v, CTL, 0xf, 0xf, true);
}
// f over the L = 32 or 64 lanes of a row: every lane ends with the result (f commutative and associative).
template <int L, typename F>
__device__ __forceinline__ uint32_t row_all(uint32_t v, F f) {
    v = f(v, dpp<0xB1>(v));   // quad_perm 1,0,3,2
    v = f(v, dpp<0x4E>(v));   // quad_perm 2,3,0,1
    v = f(v, dpp<0x141>(v));  // row_half_mirror
    v = f(v, dpp<0x140>(v));  // row_mirror
    const auto a = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    v = f((uint32_t)a[0], (uint32_t)a[1]);
    if constexpr (L == 64) {
        const auto b = __builtin_amdgcn_permlane32_swap(v, v, false, false);
        v = f((uint32_t)b[0], (uint32_t)b[1]);
    }
    return v;
}
template <int L>
__device__ __forceinline__ uint32_t row_max(uint32_t v) {
    return row_all<L>(v, [](uint32_t a, uint32_t b) { return a > b ? a : b; });
}
template <int L>
__device__ __forceinline__ double row_sum(double v) {
#pragma unroll
    for (int m = 1; m < L; m <<= 1) v = v + __shfl_xor(v, m, 64);
    return v;
}
__device__ __forceinline__ uint64_t read_lane(uint64_t u, int lane) {
    const uint32_t lo = __builtin_amdgcn_readlane((uint32_t)u, lane), hi = __builtin_amdgcn_readlane((uint32_t)(u >> 32), lane);
    return (uint64_t)lo | (uint64_t)hi << 32;
}
// What one lane of a wave wrote to LDS before is there for the others: LDS works in order, the compiler has to as well.
__device__ __forceinline__ void wave_fence() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// 1 / (1 + exp(-x)) in 64 bits: v_rcp_f64's estimate and two Newton steps (an IEEE division takes twice the instructions).
// Below -709.7827 exp(-x) is no number any more: scores end at that one's, 5.6e-309.
__device__ __forceinline__ double sigmoid64(double x) {
    const double d = 1.0 + exp(__builtin_fmin(-x, 709.7827));
    double r = __builtin_amdgcn_rcp(d);
    r = __builtin_fma(r, __builtin_fma(-d, r, 1.0), r);
    r = __builtin_fma(r, __builtin_fma(-d, r, 1.0), r);
    return x != x ? x : r;
}

// L lanes take a row, lane l its experts l, l + L, .. (EPL of them); a wave has 64 / L rows. What bounds it are instructions
// and their latencies, not bytes (256 experts x 4096 rows are 4.5 MB, 0.9 us): a 64-bit sigmoid of each logit, then the slots
// in turn, a row's largest key found by its upper half first, which only ties to 20 bits follow with the lower half and the
// expert's number. A wave a row has the shortest chain; 32 lanes a row share the steps over the lanes between two rows, which
// pays when every SIMD has several waves anyway. 256 experts, 8 slots, kernel times, 64 and 32 lanes: 1 row 4.6 us, 512 rows
// 5.3 and 6.7, 2048 rows 6.2 and 6.8, 4096 rows 8.4 and 7.8 (16 lanes took 9.8 at any of these). The loads of a row had been
// behind conditions, waited for one by one: 1 row 5.6 us, 4096 rows 12.3 then.
template <int EPL, int L, bool GROUPS>
__global__ void __launch_bounds__(256) route_kernel(RouteArgs a) {
    constexpr int ROWS = 256 / L;
    __shared__ double score[ROWS][EPL * L];
    __shared__ int32_t got[ROWS][32];
    __shared__ uint64_t keys[GROUPS ? ROWS : 1][GROUPS ? EPL * L : 1];
    const int lane = threadIdx.x & 63, l = threadIdx.x % L, w = threadIdx.x / L;
    if (blockIdx.x * (uint32_t)ROWS + (threadIdx.x & ~63u) / L >= a.rows) return;  // a whole wave; no barrier below
    const uint32_t row = min(blockIdx.x * (uint32_t)ROWS + w, a.rows - 1);  // lanes past the last row repeat it
    float x[EPL], bias[EPL];
    uint64_t key[EPL];
    {  // every load before the first use (experts past the last re-read it)
        const size_t at = (size_t)row * a.stride;
        if (a.dtype == F32) {
#pragma unroll
            for (int j = 0; j < EPL; ++j) x[j] = static_cast<const float*>(a.logits)[at + min(l + L * j, a.experts - 1)];
        } else {
            uint16_t h[EPL];
#pragma unroll
            for (int j = 0; j < EPL; ++j) h[j] = static_cast<const uint16_t*>(a.logits)[at + min(l + L * j, a.experts - 1)];
#pragma unroll
            for (int j = 0; j < EPL; ++j) x[j] = a.dtype == BF16 ? bf2f(h[j]) : h2f(h[j]);
        }
        if (a.bias) {
#pragma unroll
            for (int j = 0; j < EPL; ++j) bias[j] = a.bias[min(l + L * j, a.experts - 1)];
        } else {
#pragma unroll
            for (int j = 0; j < EPL; ++j) bias[j] = 0.0f;
        }
#pragma unroll
        for (int j = 0; j < EPL; ++j) x[j] = l + L * j < a.experts ? x[j] : -__builtin_inff();
    }
    got[w][l % 32] = -1;
    double m = 0.0, part = 0.0;
    if (a.softmax) {
        uint32_t top = 0;
#pragma unroll
        for (int j = 0; j < EPL; ++j) top = max(top, order_key(x[j]));
        top = row_max<L>(top);  // of the numbers: a NaN makes the sum NaN by itself
        const float t = __builtin_bit_cast(float, (top & 0x80000000u) ? top & 0x7fffffffu : ~top);
        m = top <= 1 || t == -__builtin_inff() ? 0.0 : (double)t;
    }
    double s[EPL];
    if (a.softmax) {
#pragma unroll
        for (int j = 0; j < EPL; ++j) {
            s[j] = exp((double)x[j] - m);
            part += s[j];
        }
        const double r = 1.0 / row_sum<L>(part);
#pragma unroll
        for (int j = 0; j < EPL; ++j) s[j] = s[j] * r;
    } else {
#pragma unroll
        for (int j = 0; j < EPL; ++j) s[j] = sigmoid64((double)x[j]);
    }
#pragma unroll
    for (int j = 0; j < EPL; ++j) {
        score[w][l + L * j] = s[j];
        key[j] = x[j] == -__builtin_inff() ? 0ull : choice_key(a.bias ? s[j] + (double)bias[j] : s[j]);
    }
    if constexpr (GROUPS) {
        static_assert(L == 64, "a group's lanes are read across the wave");
        const int size = a.experts / a.groups;
#pragma unroll
        for (int j = 0; j < EPL; ++j) keys[w][l + L * j] = key[j];
        wave_fence();
        // per neighbouring lanes (a power of two) rank a group by the sum of its one or two best choices, those it has
        const int per = 1 << (31 - __builtin_clz(64 / a.groups)), g = lane / per;
        uint64_t first = 0, second = 0;
        for (int i = lane % per; g < a.groups && i < size; i += per) {
            const uint64_t k = keys[w][g * size + i];
            second = k > first ? first : k > second ? k : second;
            first = k > first ? k : first;
        }
        for (int d = 1; d < per; d <<= 1) {
            const uint64_t of = __shfl_xor(first, d, 64), os = __shfl_xor(second, d, 64), s2 = os > second ? os : second;
            const uint64_t lo = of > first ? first : of;
            second = lo > s2 ? lo : s2;
            first = of > first ? of : first;
        }
        uint64_t rank = first;
        if (a.group_best == 2 && second) rank = choice_key(choice_of(first) + choice_of(second));
        int before = 0;
        for (int o = 0; o < a.groups; ++o) {
            const uint64_t r = read_lane(rank, o * per);
            before += r > rank || (r == rank && o < g);
        }
        const uint64_t kept = __ballot(g < a.groups && before < a.top_groups);  // bit per * g
#pragma unroll
        for (int j = 0; j < EPL; ++j) {
            const int e = l + L * j;
            if (e < a.experts && !(kept >> (e / size * per) & 1)) key[j] = 0;
        }
    }
    wave_fence();
    // the slots in turn
    const auto row_bits = [&](uint64_t b) { return L == 64 ? b : b >> (lane & ~(L - 1)) & ((1ull << (L & 63)) - 1); };
    for (int k = 0; k < a.slots; ++k) {
        uint64_t best = key[0];
        int at = l;
#pragma unroll
        for (int j = 1; j < EPL; ++j) {
            const bool more = key[j] > best;
            best = more ? key[j] : best;
            at = more ? l + L * j : at;
        }
        const uint32_t hi = (uint32_t)(best >> 32), top = row_max<L>(hi);
        bool win = hi == top && best != 0;
        const uint64_t tied = row_bits(__ballot(win));
        if (__ballot((tied & (tied - 1)) != 0)) {  // equal upper halves in some row
            const uint32_t lo = win ? (uint32_t)best : 0, ltop = row_max<L>(lo);
            win = win && lo == ltop;
            const uint32_t last = row_max<L>(win ? 0xffffffffu - at : 0);
            win = win && 0xffffffffu - at == last;
        }
        if (win) got[w][k] = at;
#pragma unroll
        for (int j = 0; j < EPL; ++j) key[j] = win && at == l + L * j ? 0 : key[j];
    }
    wave_fence();
    double sum = 0.0;
    if (a.renorm) {
        for (int k = l; k < a.slots; k += L) sum += got[w][k] < 0 ? 0.0 : score[w][got[w][k]];
        sum = row_sum<L>(sum) + 1e-20;
    }
    if (blockIdx.x * (uint32_t)ROWS + w >= a.rows) return;
    for (int k = l; k < a.slots; k += L) {
        const int e = got[w][k];
        const double v = e < 0 ? 0.0 : a.renorm ? score[w][e] / sum : score[w][e];
        a.pick[(size_t)row * a.slots + k] = e;
        a.wts[(size_t)row * a.slots + k] = (float)(v * (double)a.scale);
    }
}

static int launch_route(hipStream_t s, const RouteArgs& a) {
    auto go = [&](auto epl) {
        constexpr int EPL = decltype(epl)::value;
        if (a.groups > 1) route_kernel<EPL, 64, true><<<(a.rows + 3) / 4, 256, 0, s>>>(a);
        else if (EPL > 4 || a.rows < 4096) route_kernel<EPL, 64, false><<<(a.rows + 3) / 4, 256, 0, s>>>(a);
        else route_kernel<2 * std::min(EPL, 4), 32, false><<<(a.rows + 7) / 8, 256, 0, s>>>(a);
    };
    if (a.experts <= 64) go(std::integral_constant<int, 1>{});
    else if (a.experts <= 128) go(std::integral_constant<int, 2>{});
    else if (a.experts <= 256) go(std::integral_constant<int, 4>{});
    else if (a.experts <= 512) go(std::integral_constant<int, 8>{});
    else go(std::integral_constant<int, 16>{});
    return launched();
}

}  // namespace ea

extern "C" int ea_route(ea_stream_t stream, const void* logits, int l_dtype, uint32_t l_stride, const float* bias,
                        int32_t* pick, float* wts, uint32_t rows, uint32_t experts, uint32_t slots, int score,
                        uint32_t groups, uint32_t top_groups, uint32_t group_best, int renorm, float scale) {
    using namespace ea;
    if (!logits || !pick || !wts || l_dtype < F16 || l_dtype > F32) return EA_BAD_ARGUMENT;
    if (score != EA_SCORE_SIGMOID && score != EA_SCORE_SOFTMAX) return EA_BAD_ARGUMENT;
    if (experts == 0 || slots == 0) return EA_BAD_ARGUMENT;
    if (experts > EA_ROUTE_MAX_EXPERTS) return EA_TOO_MANY_EXPERTS;
    if (slots > 32) return EA_TOO_MANY_SLOTS;
    if (l_stride < experts) return EA_BAD_ROW_STRIDE;
    if (groups == 0 || groups > 64 || top_groups == 0 || top_groups > groups || group_best < 1 || group_best > 2)
        return EA_BAD_ARGUMENT;
    if (experts % groups != 0) return EA_UNEVEN_SPLIT;
    if (slots > experts / groups * top_groups) return EA_TOO_MANY_SLOTS;
    EA_REQUIRE_CTX(ctx_);
    (void)ctx_;
    if (rows == 0) return EA_OK;
    RouteArgs a{logits, bias, pick, wts, l_stride, rows, (int)experts, (int)slots, (int)groups, (int)top_groups,
                (int)group_best, l_dtype, score == EA_SCORE_SOFTMAX, renorm != 0, scale};
    return launch_route(as_stream(stream), a);
}
