// Routing to experts in its general form: softmax or sigmoid scores, a bias for balance that takes part in the choice alone,
// groups of experts of which the best are kept, the k largest choices, weights that are renormalised and scaled.
//
// A choice is compared in 64 bits: the picks are whole numbers, two choices can lie closer than a 32-bit sigmoid's error, and
// a balance bias moves them to within it on purpose, so that the picks would otherwise depend on how a sigmoid rounds. A
// wave takes a row, lane l its experts l, l + 64, ..
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

template <int M, typename T>
__device__ __forceinline__ T lane_xor64(T v) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const float lo = lane_xor<M>(__builtin_bit_cast(float, (uint32_t)u));
    const float hi = lane_xor<M>(__builtin_bit_cast(float, (uint32_t)(u >> 32)));
    return __builtin_bit_cast(T, (uint64_t)__builtin_bit_cast(uint32_t, lo) | (uint64_t)__builtin_bit_cast(uint32_t, hi) << 32);
}

// f over the wave by the butterfly: every lane ends with the same value.
template <typename T, typename F>
__device__ __forceinline__ T wave_all(T v, F f) {
    v = f(v, lane_xor64<32>(v));
    v = f(v, lane_xor64<16>(v));
    v = f(v, lane_xor64<8>(v));
    v = f(v, lane_xor64<4>(v));
    v = f(v, lane_xor64<2>(v));
    return f(v, lane_xor64<1>(v));
}

__device__ __forceinline__ double read_lane(double v, int lane) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = __builtin_amdgcn_readlane((uint32_t)u, lane), hi = __builtin_amdgcn_readlane((uint32_t)(u >> 32), lane);
    return __builtin_bit_cast(double, (uint64_t)lo | (uint64_t)hi << 32);
}

constexpr int ROUTE_WAVES = 4;

template <int EPL, bool GROUPS>
__global__ void __launch_bounds__(64 * ROUTE_WAVES) route_kernel(RouteArgs a) {
    __shared__ uint64_t keys[GROUPS ? ROUTE_WAVES : 1][GROUPS ? 64 * EPL : 1];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint32_t row = blockIdx.x * ROUTE_WAVES + wave;
    if (row >= a.rows) return;  // no barrier below: a wave works alone
    float x[EPL];
    double s[EPL];
    uint64_t key[EPL];
#pragma unroll
    for (int j = 0; j < EPL; ++j) {
        const int e = lane + 64 * j;
        x[j] = e < a.experts ? load_act(a.logits, a.dtype, (size_t)row * a.stride + e) : -__builtin_inff();
    }
    if (a.softmax) {
        float top = x[0];
#pragma unroll
        for (int j = 1; j < EPL; ++j) top = __builtin_fmaxf(top, x[j]);
        const double m = wave_all((double)top, [](double p, double q) { return __builtin_fmax(p, q); });
        const double m0 = m == -__builtin_inf() ? 0.0 : m;
        double sum = 0.0;
#pragma unroll
        for (int j = 0; j < EPL; ++j) {
            s[j] = exp((double)x[j] - m0);
            sum += s[j];
        }
        sum = wave_all(sum, [](double p, double q) { return p + q; });
#pragma unroll
        for (int j = 0; j < EPL; ++j) s[j] = s[j] / sum;
    } else {
#pragma unroll
        for (int j = 0; j < EPL; ++j) s[j] = 1.0 / (1.0 + exp(-(double)x[j]));
    }
#pragma unroll
    for (int j = 0; j < EPL; ++j) {
        const int e = lane + 64 * j;
        const double c = a.bias && e < a.experts ? s[j] + (double)a.bias[e] : s[j];
        key[j] = x[j] == -__builtin_inff() ? 0ull : choice_key(c);
    }
    if constexpr (GROUPS) {
        const int size = a.experts / a.groups;
#pragma unroll
        for (int j = 0; j < EPL; ++j) keys[wave][lane + 64 * j] = key[j];
        __builtin_amdgcn_wave_barrier();
        // lane g ranks group g by the sum of its one or two best choices (those that it has)
        uint64_t first = 0, second = 0;
        if (lane < a.groups)
            for (int i = 0; i < size; ++i) {
                const uint64_t k = keys[wave][lane * size + i];
                second = k > first ? first : k > second ? k : second;
                first = k > first ? k : first;
            }
        uint64_t rank = first;
        if (a.group_best == 2 && second) rank = choice_key(choice_of(first) + choice_of(second));
        int before = 0;
        for (int g = 0; g < a.groups; ++g) {
            const uint64_t o = __builtin_bit_cast(uint64_t, read_lane(__builtin_bit_cast(double, rank), g));
            before += o > rank || (o == rank && g < lane);
        }
        const uint64_t kept = __ballot(lane < a.groups && before < a.top_groups);
#pragma unroll
        for (int j = 0; j < EPL; ++j) {
            const int e = lane + 64 * j;
            if (e < a.experts && !(kept >> (e / size) & 1)) key[j] = 0;
        }
    }
    // the slots in turn: the largest key of the wave, the lowest expert that holds it
    double sum = 0.0, mine = 0.0;
    int mine_e = -1;
    for (int k = 0; k < a.slots; ++k) {
        uint64_t best = key[0];
#pragma unroll
        for (int j = 1; j < EPL; ++j) best = key[j] > best ? key[j] : best;
        best = wave_all(best, [](uint64_t p, uint64_t q) { return p > q ? p : q; });
        if (best == 0) break;  // none left: this slot and the ones after it stay empty
        int at = -1, who = 0;
        double w = 0.0;
#pragma unroll
        for (int j = EPL - 1; j >= 0; --j) {
            const uint64_t has = __ballot(key[j] == best);
            if (has) {
                who = __builtin_ctzll(has);
                at = who + 64 * j;
                w = read_lane(s[j], who);
            }
        }
#pragma unroll
        for (int j = 0; j < EPL; ++j) key[j] = at == lane + 64 * j ? 0 : key[j];
        sum += w;
        if (lane == k) {
            mine = w;
            mine_e = at;
        }
    }
    if (lane < a.slots) {
        const size_t o = (size_t)row * a.slots + lane;
        const double w = mine_e < 0 ? 0.0 : a.renorm ? mine / (sum + 1e-20) : mine;
        a.pick[o] = mine_e;
        a.wts[o] = (float)(w * (double)a.scale);
    }
}

static int launch_route(hipStream_t s, const RouteArgs& a) {
    const unsigned blocks = (a.rows + ROUTE_WAVES - 1) / ROUTE_WAVES;
    auto go = [&](auto epl) {
        constexpr int EPL = decltype(epl)::value;
        if (a.groups > 1) route_kernel<EPL, true><<<blocks, 64 * ROUTE_WAVES, 0, s>>>(a);
        else route_kernel<EPL, false><<<blocks, 64 * ROUTE_WAVES, 0, s>>>(a);
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
