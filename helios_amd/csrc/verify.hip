// Drafted tokens checked against the target's probabilities, and tokens sampled from logits.
//
//   z_i = cap tanh(x_i / cap) / T,  p_i = e^(z_i) / sum_j e^(z_j)   (q likewise of the drafter's)
//   draft d, the token of the next row, stands while u q_d < p_d
//   the first that does not: a token from max(p - q, 0); all stand: one from the last row's p
//   from weights w: the first i with w_0 + .. + w_i > u (w_0 + .. + w_(n-1))
//   T = 0: p and q are 1 at the first largest logit, 0 elsewhere
//   a logit of -inf or NaN, and a weight under e^-700 of the largest, is 0 whatever cap and T; a drafter that
//   gives no logits is sure (q_d = 1)
//
// Sums and weights are fp64: a token is a place in a sum of some 2^18 terms, and an fp32 sum
// (2^-24 of it off) would miss by one wherever the terms are smaller than that.
//
// Bound by reading the logits once, and as much by their exponentials: twelve operations each, nine of
// them fp64, of 4.2 to 4.5 cycles a wave.  A row is cut into parts of 2048 (or 512) places; a wave holds
// a part in registers between the search for its maximum and the sum of its weights relative to
// that (stats_kernel).  Each request's own workgroups then join its rows' sums, find the first
// draft that falls and sum max(p - q, 0) over parts of that one row (rest_kernel); a workgroup per
// request finds the part and the place in it (pick_kernel).  Orders are fixed: no atomics.
//
// us of the three, rows of 262144: 32 requests of 8 rows, bf16, with the drafter's rows (252 MB) 80 + 18 +
// 7 (3.2 TB/s in the first, whose 31M operations are 53 us of issue); 256 rows without drafts (134 MB) 38 + 6, capped 84 in all;
// 48 rows of fp32 (50 MB) 13 + 5 (3.8 TB/s); one row 3.7 + 6, two launches and a chain of loads.
// Parts one after another in a wave, the next one's loads ahead of this one's sums: 84 for the 80.
#include "q4_common.h"
#include "verify_index.h"
#include "verify_kernels.h"

// rest_kernel and pick_kernel weigh the same places and have to agree on them to the last bit
#pragma clang fp contract(off)

namespace verify {
namespace {

// The sum of a part's weights relative to `top`, the largest logit (as it is) of the part's
// chunk; for greedy requests the first place that has it.
struct alignas(16) Part {
    double sum;
    float top;
    int at;
};

// What a request's row to sample from is: written by rest_kernel, read by pick_kernel.
struct alignas(16) Spot {
    double p_scale, q_scale;  // weights e^(..) times these are p and q
    float p_top, q_top;
    int row, token;           // token: the draft that fell where the drafter is sure; -1: none
    int kind;                 // 0: nothing to sample, 1: from p, 2: from max(p - q, 0)
    int pad;
};

struct Work {
    Part* parts;   // [target rows, then drafter's rows][parts]
    double* rest;  // [requests][parts], of requests whose spot is of kind 2
    Spot* spots;   // [requests]
};

__device__ __forceinline__ int clampi(int v, int lo, int hi) { return v < lo ? lo : (v > hi ? hi : v); }
constexpr float kInf = __builtin_huge_valf();

// 2^(j / 256), by the series of the exponential; j / 256 is taken off the exponent and mantissa
// field again, so that adding n 2^-8 to that field, n % 256 = j, gives the bits of 2^(n / 256).
constexpr int kSteps = 256;
typedef uint32_t U2 __attribute__((ext_vector_type(2)));
struct Exp2Table {
    uint64_t v[kSteps];
};
constexpr Exp2Table make_exp2() {
    Exp2Table t{};
    for (int j = 0; j < kSteps; ++j) {
        const double x = 0.69314718055994530942 * j / kSteps;
        double sum = 0.0;
        for (int k = 24; k > 0; --k) sum = (sum + 1.0) * x / k;
        t.v[j] = __builtin_bit_cast(uint64_t, 1.0 + sum) - ((uint64_t)j << 44);
    }
    return t;
}
__device__ const Exp2Table kExp2 = make_exp2();

template <int THREADS>
__device__ __forceinline__ void take_exp2(U2* table) {
    if (THREADS == kSteps || (int)threadIdx.x < kSteps) table[threadIdx.x] = __builtin_bit_cast(U2, kExp2.v[threadIdx.x]);
}

// e^z for kLeast <= z <= 0, 2e-13 of it off at most; any bits for other z.  z = (n + r) ln2 / 256 with
// |r| <= 1/2: the series to the third power of at most ln2 / 512 (the next term is 1.4e-13), and a
// factor 2^(n / 256) from the table.  The constants sit in registers from the kernel's start.
constexpr double kLeast = -700.0;
struct Exp {
    const U2* table;
    double per_step, step, sixth, magic;
    __device__ __forceinline__ explicit Exp(const U2* t)
        : table(t), per_step(kSteps / 0.69314718055994530942), step(-0.69314718055994530942 / kSteps), sixth(1.0 / 6),
          magic(6755399441055744.0) {  // 1.5 * 2^52: the low bits of a sum with it are the nearest integer
        asm volatile("" : "+s"(per_step), "+s"(step), "+s"(sixth));
        asm volatile("" : "+v"(magic));
    }
    __device__ __forceinline__ double operator()(double z) const {
        const double t = __builtin_fma(z, per_step, magic);
        const uint32_t n = (uint32_t)__builtin_bit_cast(uint64_t, t);
        const double r = __builtin_fma(t - magic, step, z);
        U2 two = table[n & (kSteps - 1)];
        two.y += n << 12;
        const double f = __builtin_bit_cast(double, two);
        const double q = __builtin_fma(__builtin_fma(r, sixth, 0.5), r, 1.0);
        return __builtin_fma(f * r, q, f);
    }
};

__device__ __forceinline__ double lane_of(double v, int lane) {
    const uint64_t bits = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)bits, lane), hi = __builtin_amdgcn_readlane((int)(uint32_t)(bits >> 32), lane);
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}

// The larger; b where a is NaN (the compiler's own form takes two operations).
__device__ __forceinline__ double at_least(double a, double b) {
    double v;
    asm("v_max_f64 %0, %1, %2" : "=v"(v) : "v"(a), "s"(b));
    return v;
}

// A distribution over a row's places: z = cap tanh(x / cap) / T, relative to that of `top`.
struct Scale {
    double inv_heat, top;       // 1 / T
    double cap_heat, inv_cap2;  // cap / T and 2 / cap (0: no cap)
    double at_top;              // capped: z of the top or, where cap / T is over kSteep, its factor of z
};

// cap / T up to which tanh itself is taken, 1e-13 off: z is off by cap / T * 2e-13, 6e-12 at a cap of 30 and T = 1, 3e-9 at
// most.  256 rows of 262144 bf16: 84 us, and 224 past kSteep.
constexpr double kSteep = 16384.0;

__device__ __forceinline__ double reciprocal(double d) {
    double y = __builtin_amdgcn_rcp(d);
    y = __builtin_fma(__builtin_fma(-d, y, 1.0), y, y);
    return __builtin_fma(__builtin_fma(-d, y, 1.0), y, y);
}
// tanh(x / cap) by e^-2|a| of a = x / cap: 2 / (1 + e^-2|a|) - 1; the hardware's estimate is 2^-24 off, a step squares that
__device__ __forceinline__ double tanh_of(float x, double inv_cap2, const Exp& exp) {
    const double e = exp(at_least(__builtin_fabs((double)x) * -inv_cap2, kLeast)), d = 1.0 + e;
    double y = __builtin_amdgcn_rcp(d);
    y = __builtin_fma(__builtin_fma(-d, y, 1.0), y, y);
    return __builtin_copysign(__builtin_fma(2.0, y, -1.0), (double)x);
}

// Past kSteep, and with it for large caps, the difference of two tanh is formed as a product, some 5e-13 of itself off:
//   tanh a - tanh b = 2 s(-2a) (e^(2 (a - b)) - 1) s(2b),  s(v) = 1 / (1 + e^-v)
__device__ __forceinline__ double logistic(double v, const Exp& exp) {
    const double size = -__builtin_fabs(v), e = size >= kLeast ? exp(size) : 0.0, y = reciprocal(1.0 + e);
    return v < 0.0 ? e * y : y;
}
struct Inverses {
    double v[15];
};
constexpr Inverses make_inverses() {
    Inverses t{};
    for (int k = 1; k < 15; ++k) t.v[k] = 1.0 / k;
    return t;
}
__device__ const Inverses kInverse = make_inverses();
// e^v - 1 of v <= 0: the series to the 14th power (4e-17) where e^v is near 1.
__device__ __forceinline__ double exp_less_one(double v, const Exp& exp) {
    if (v < -0.5) return v >= kLeast ? exp(v) - 1.0 : -1.0;
    double sum = 1.0;
#pragma unroll 1  // in line its constants take the registers of the paths beside it
    for (int k = 14; k > 1; --k) sum = __builtin_fma(sum * v, kInverse.v[k], 1.0);
    return sum * v;
}

template <bool CAP>
__device__ __forceinline__ Scale scale_of(float top, double cap, double inv_heat, const Exp& exp) {
    Scale s{inv_heat, (double)top, cap * inv_heat, CAP && cap > 0.0 ? 2.0 / cap : 0.0, 0.0};
    if (CAP && s.inv_cap2 > 0.0)
        s.at_top = s.cap_heat > kSteep ? 2.0 * s.cap_heat * logistic(s.top * s.inv_cap2, exp) : s.cap_heat * tanh_of(top, s.inv_cap2, exp);
    return s;
}

// z relative to the top's, kLeast or less (or NaN) for -inf and NaN; the top finite, or capped and not -inf.
template <bool CAPPED>
__device__ __forceinline__ double exponent(float x, const Scale& s, const Exp& exp) {
    // x - top is exact, or off by 2^-53 of it; x / T - top / T would be off by that of a quotient without bound
    if (!CAPPED) return ((double)x - s.top) * s.inv_heat;
    const double z = __builtin_fma(tanh_of(x, s.inv_cap2, exp), s.cap_heat, -s.at_top);
    // of -inf and NaN kLeast's upper half, with any lower one
    const U2 least = __builtin_bit_cast(U2, kLeast);
    U2 bits = __builtin_bit_cast(U2, z);
    bits.y = x > -kInf ? bits.y : least.y;
    return __builtin_bit_cast(double, bits);
}
// e^(z(x) - z(top)); 0 for -inf, NaN and less than e^-700; x is not over the top.
template <bool CAP>
__device__ __forceinline__ double weight(float x, const Scale& s, const Exp& exp) {
    if (CAP && s.inv_cap2 > 0.0) {
        const double z = s.cap_heat > kSteep ? s.at_top * logistic((double)x * -s.inv_cap2, exp) * exp_less_one(((double)x - s.top) * s.inv_cap2, exp)
                                             : exponent<true>(x, s, exp);
        const double e = z >= kLeast ? exp(z) : 0.0;
        return x == kInf ? 1.0 : (x > -kInf ? e : 0.0);
    }
    const double z = exponent<false>(x, s, exp), e = z >= kLeast ? exp(z) : 0.0;
    return x == kInf ? 1.0 : e;  // beside infinity nothing finite has a weight
}
// The weight as a term of a sum, where e^-700 is nothing.
template <bool CAPPED>
__device__ __forceinline__ double term(float x, const Scale& s, const Exp& exp) {
    return exp(at_least(exponent<CAPPED>(x, s, exp), kLeast));
}

// Sums of uncapped terms with two operations less than term's, the same shape of e^z in x's own
// units: x = (N + r) T ln2 / 256, N's share of the top taken off in t, r's at the end.
struct Sum {
    const U2* table;
    double a, b, step, c1, c2, c3, least, sum;
    // |top / T| under 2^40, so that N has room
    __device__ __forceinline__ Sum(const Exp& exp, float top, double inv_heat, double heat)
        : table(exp.table), a(inv_heat * exp.per_step), step(heat * exp.step), c1(inv_heat), c2(0.5 * inv_heat * inv_heat),
          c3(inv_heat * inv_heat * inv_heat * exp.sixth), least(__builtin_fma(heat, kLeast, (double)top)), sum(0.0) {
        b = exp.magic - (__builtin_fma((double)top, a, exp.magic) - exp.magic);
        // the wave's own: to scalar registers, of which an operation takes one
        a = lane_of(a, 0), step = lane_of(step, 0), c1 = lane_of(c1, 0), c3 = lane_of(c3, 0), least = lane_of(least, 0);
    }
    __device__ __forceinline__ double series(double r) const {
        return __builtin_fma(__builtin_fma(__builtin_fma(r, c3, c2), r, c1), r, 1.0);
    }
    __device__ __forceinline__ void add(float logit) {
        const double x = at_least((double)logit, least), t = __builtin_fma(x, a, b);
        const uint32_t n = (uint32_t)__builtin_bit_cast(uint64_t, t);
        U2 two = table[n & (kSteps - 1)];
        two.y += n << 12;
        sum = __builtin_fma(__builtin_bit_cast(double, two), series(__builtin_fma(t - b, step, x)), sum);
    }
    __device__ __forceinline__ double relative_to(float top, const Exp& exp) const {
        return sum * series(-__builtin_fma(exp.magic - b, step, (double)top));
    }
};
constexpr double kRoomy = 0x1p40;

template <bool CAP>
__device__ __forceinline__ double any_term(float x, const Scale& s, const Exp& exp) {
    return CAP && s.inv_cap2 > 0.0 ? term<true>(x, s, exp) : term<false>(x, s, exp);
}

// Eight logits from place i0 on, as they are; -inf from `end` on.
template <bool F32>
__device__ __forceinline__ void load8(const Logits& l, int64_t row, int i0, int end, uint32_t (&w)[F32 ? 8 : 4]) {
    typedef uint32_t U4 __attribute__((ext_vector_type(4), aligned(2)));  // rows may start anywhere
    const int64_t at = row * l.stride + i0;
    if (i0 + 8 <= end) {
        const U4* const from = reinterpret_cast<const U4*>(static_cast<const char*>(l.x) + at * (F32 ? 4 : 2));
#pragma unroll
        for (int j = 0; j < (F32 ? 2 : 1); ++j) {
            const U4 v = from[j];
#pragma unroll
            for (int i = 0; i < 4; ++i) w[4 * j + i] = v[i];
        }
        return;
    }
    if constexpr (F32) {
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = i0 + i < end ? static_cast<const uint32_t*>(l.x)[at + i] : 0xFF800000u;
    } else {
        const auto one = [&](int i) { return i0 + i < end ? (uint32_t) static_cast<const uint16_t*>(l.x)[at + i] : 0xFF80u; };
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = one(2 * i) | one(2 * i + 1) << 16;
    }
}
template <bool F32>
__device__ __forceinline__ float load1(const Logits& l, int64_t row, int at) {
    const int64_t i = row * l.stride + at;
    return F32 ? static_cast<const float*>(l.x)[i] : __uint_as_float((uint32_t) static_cast<const uint16_t*>(l.x)[i] << 16);
}

template <int DPP, int ROWS>
__device__ __forceinline__ double dpp_of(double v) {
    const uint64_t bits = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)bits, DPP, ROWS, 0xf, ROWS == 0xf);
    const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)(bits >> 32), DPP, ROWS, 0xf, ROWS == 0xf);
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
// Inclusive sums over the lanes (row shifts of 1, 2, 4, 8, then the rows' last lanes to the rows after
// them), and the sum of all.
__device__ __forceinline__ double wave_scan(double v) {
    v += dpp_of<0x111, 0xf>(v);
    v += dpp_of<0x112, 0xf>(v);
    v += dpp_of<0x114, 0xf>(v);
    v += dpp_of<0x118, 0xf>(v);
    v += dpp_of<0x142, 0xa>(v);
    v += dpp_of<0x143, 0xc>(v);
    return v;
}
__device__ __forceinline__ double wave_sum(double v) { return lane_of(wave_scan(v), 63); }
template <int DPP, int ROWS>
__device__ __forceinline__ float dpp_top(float v) {
    return fmaxf(v, __int_as_float(__builtin_amdgcn_update_dpp(__float_as_int(v), __float_as_int(v), DPP, ROWS, 0xf, false)));
}
__device__ __forceinline__ float wave_top(float v) {
    v = dpp_top<0x118, 0xf>(dpp_top<0x114, 0xf>(dpp_top<0x112, 0xf>(dpp_top<0x111, 0xf>(v))));
    v = dpp_top<0x143, 0xc>(dpp_top<0x142, 0xa>(v));
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 63));
}
__device__ __forceinline__ int wave_least(int v) {
#pragma unroll
    for (int d = 32; d > 0; d /= 2) {
        const int o = __shfl_xor(v, d);
        v = o < v ? o : v;
    }
    return v;
}

// The request of a row; `requests` for none.  Every lane of the wave takes part.
__device__ __forceinline__ int request_of(const Args& a, int row) {
    if (a.starts == nullptr) return row;
    const int lane = (int)threadIdx.x & 63;
    int request = 0;
    for (int base = 0; base < a.requests; base += 64) {
        const int i = base + lane;
        const int end = i < a.requests ? a.starts[i + 1] : 0x7fffffff;
        const unsigned long long past = __ballot(end <= row);
        request += __popcll(past);
        if (past != ~0ull) break;
    }
    return row < a.starts[0] ? a.requests : request;
}
__device__ __forceinline__ int start_of(const Args& a, int r) { return a.starts == nullptr ? r : clampi(a.starts[r], 0, a.rows); }
// The request's temperature; 0 where it is greedy.  For infinity 1e60, over which all logits are equal.
__device__ __forceinline__ double heat_of(const Args& a, int r) {
    const float t = a.heats != nullptr ? a.heats[r] : a.heat;
    return t > 0.0f ? (t < kInf ? (double)t : 1e60) : 0.0;
}
__device__ __forceinline__ double inv_of(double heat) { return heat > 0.0 ? 1.0 / heat : 0.0; }
__device__ __forceinline__ double inv_heat_of(const Args& a, int r) { return inv_of(heat_of(a, r)); }

constexpr int kNowhere = 0x7fffffff;

// A part's logits as a wave holds them: lane l has places 512 j + 8 l + i (j < S, i < 8).
template <bool F32, int S>
struct Held {
    uint32_t w[S][F32 ? 8 : 4];
    __device__ __forceinline__ void load(const Logits& l, int64_t row, int begin, int vocab) {
        const int lane = (int)threadIdx.x & 63;
#pragma unroll
        for (int j = 0; j < S; ++j) load8<F32>(l, row, begin + 512 * j + 8 * lane, vocab, w[j]);
    }
    __device__ __forceinline__ float at(int j, int i) const {
        if (F32) return __uint_as_float(w[j][i]);
        return __uint_as_float((i & 1) ? w[j][i / 2] & 0xFFFF0000u : w[j][i / 2] << 16);
    }
};

template <bool F32, bool CAP, int S>
__global__ __launch_bounds__(kStatsThreads, F32 && S > 1 ? 5 : 8) void stats_kernel(Args a, Work w, Plan plan) {
    __shared__ U2 table[kSteps];
    const int lane = (int)threadIdx.x & 63;
    const Place place = place_of(plan, __builtin_amdgcn_readfirstlane((int)blockIdx.x * (kStatsThreads / 64) + ((int)threadIdx.x >> 6)));
    const bool of_draft = place.row >= a.rows;  // the plan has those rows only where there is a drafter
    const int row = of_draft ? place.row - a.rows : place.row;
    const Logits& l = of_draft ? a.draft : a.target;
    const int begin = place.part * plan.size();
    Held<F32, S> x;
    if (place.part >= 0) x.load(l, row, begin, a.vocab);
    take_exp2<kStatsThreads>(table);
    const Exp exp(table);
    __syncthreads();
    if (place.part < 0) return;
    const int r = request_of(a, row);
    if (r >= a.requests) return;                                // padding
    if (of_draft && row + 1 >= start_of(a, r + 1)) return;      // no draft was drawn from it
    const double heat = heat_of(a, r), inv_heat = inv_of(heat);
    float top = -kInf;
#pragma unroll
    for (int j = 0; j < S; ++j)
#pragma unroll
        for (int i = 0; i < 8; ++i) top = fmaxf(top, x.at(j, i));  // NaN has no say
    top = wave_top(top);
    double sum = 0.0;
    int at = kNowhere;
    if (inv_heat > 0.0) {
        const Scale scale = scale_of<CAP>(top, l.cap, inv_heat, exp);
        const bool capped = CAP && scale.inv_cap2 > 0.0;
        if (capped && top > -kInf && scale.cap_heat <= kSteep) {
#pragma unroll
            for (int j = 0; j < S; ++j)
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    sum += term<true>(x.at(j, i), scale, exp);
                    if (i == 7) __builtin_amdgcn_sched_barrier(0);
                }
        } else if (!capped && __builtin_fabs((double)top * inv_heat) < kRoomy) {
            Sum of(exp, top, inv_heat, heat);
#pragma unroll
            for (int j = 0; j < S; ++j)
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    of.add(x.at(j, i));
                    if (i == 7) __builtin_amdgcn_sched_barrier(0);  // more at once do not fit the registers
                }
            sum = of.relative_to(top, exp);
        } else {  // nothing, infinities (which share all there is), larger than Sum has room for, or past kSteep
            const int end = begin + 512 * S < a.vocab ? begin + 512 * S : a.vocab;
            for (int i = begin + lane; i < end; i += 64) sum += weight<CAP>(load1<F32>(l, row, i), scale, exp);
        }
        sum = wave_sum(sum);
    } else if (top > -kInf) {
#pragma unroll
        for (int j = S - 1; j >= 0; --j)
#pragma unroll
            for (int i = 7; i >= 0; --i) at = x.at(j, i) == top ? begin + 512 * j + 8 * lane + i : at;
        at = wave_least(at);
    }
    if (lane == 0) w.parts[(int64_t)place.row * plan.parts + place.part] = Part{sum, top, at};
}

struct Total {
    double sum;
    float top;
    int at;
};
// A row's parts joined, by the lanes of a wave.
template <bool CAP, int HELD>
__device__ __forceinline__ Total join(const Part* parts, int count, double cap, double inv_heat, const Exp& exp) {
    const int lane = (int)threadIdx.x & 63;
    Total t{0.0, -kInf, kNowhere};
    const Part none{0.0, -kInf, kNowhere};
    // the first of a lane's parts stay in registers
    constexpr int kHeld = HELD;
    Part held[kHeld];
#pragma unroll
    for (int i = 0; i < kHeld; ++i) held[i] = lane + 64 * i < count ? parts[lane + 64 * i] : none;
#pragma unroll
    for (int i = 0; i < kHeld; ++i) t.top = fmaxf(t.top, held[i].top);
    for (int i = lane + 64 * kHeld; i < count; i += 64) t.top = fmaxf(t.top, parts[i].top);
    t.top = wave_top(t.top);
    if (inv_heat > 0.0) {
        const Scale scale = scale_of<CAP>(t.top, cap, inv_heat, exp);
#pragma unroll
        for (int i = 0; i < kHeld; ++i) t.sum += held[i].sum * weight<CAP>(held[i].top, scale, exp);
        for (int i = lane + 64 * kHeld; i < count; i += 64) t.sum += parts[i].sum * weight<CAP>(parts[i].top, scale, exp);
        t.sum = wave_sum(t.sum);
    } else {
#pragma unroll
        for (int i = 0; i < kHeld; ++i)
            if (held[i].top == t.top) t.at = held[i].at < t.at ? held[i].at : t.at;
        for (int i = lane + 64 * kHeld; i < count; i += 64)
            if (parts[i].top == t.top) t.at = parts[i].at < t.at ? parts[i].at : t.at;
        t.at = wave_least(t.at);
    }
    return t;
}

// The weight of place `at` (-1: none), whose logit is x, in a row of that total; greedy: 1 at its first
// largest logit.
template <bool CAP>
__device__ __forceinline__ double weight_at(const Logits& l, int at, float x, const Total& t, double inv_heat, const Exp& exp) {
    if (at < 0) return 0.0;
    if (!(inv_heat > 0.0)) return at == t.at ? 1.0 : 0.0;
    return weight<CAP>(x, scale_of<CAP>(t.top, l.cap, inv_heat, exp), exp);
}

// The weights of a request's row to sample from.
template <bool CAP>
struct Rest {
    Scale p, q;
    double p_scale, q_scale;
    int token;
    bool minus_q;
    __device__ __forceinline__ Rest(const Args& a, const Spot& s, double inv_heat, const Exp& exp)
        : p(scale_of<CAP>(s.p_top, a.target.cap, inv_heat, exp)), p_scale(s.p_scale), q_scale(s.q_scale), token(s.token),
          minus_q(s.kind == 2 && a.draft.x != nullptr) {
        q = minus_q ? scale_of<CAP>(s.q_top, a.draft.cap, inv_heat, exp) : p;
        const auto holds = [](float top, const Scale& z) { return CAP && z.inv_cap2 > 0.0 ? top > -kInf && z.cap_heat <= kSteep : fabsf(top) < kInf; };
        plain = holds(s.p_top, p) && (!minus_q || holds(s.q_top, q));
        nothing = exp(kLeast);
    }
    // Whether exponent() holds of both.
    bool plain;
    double nothing;  // the term of a place without weight
    // Place `at`, whose logit is x and the drafter's y; PLAIN: with an operation or two less, within its error of
    // what the other gives.  A part summed by one of them is searched by the same one, so that its sum is over
    // zero exactly where one of its places has a weight (p - q can be nothing but such differences).
    template <bool PLAIN>
    __device__ __forceinline__ double of(int at, float x, float y, const Exp& exp) const {
        double v;
        if (PLAIN) {
            v = (any_term<CAP>(x, p, exp) - nothing) * p_scale;  // changes no term over 1e-288; of q's it may stay
            if (minus_q) v = __builtin_fmax(__builtin_fma(-any_term<CAP>(y, q, exp), q_scale, v), 0.0);
        } else {
            v = weight<CAP>(x, p, exp) * p_scale;
            if (minus_q) v = __builtin_fmax(__builtin_fma(-weight<CAP>(y, q, exp), q_scale, v), 0.0);
        }
        return at == token ? 0.0 : v;
    }
};

// A row's total as what to sample from it.
__device__ __forceinline__ Spot spot_of(const Total& p, int row, double inv_heat, int kind) {
    Spot s{};
    s.row = row;
    s.kind = inv_heat > 0.0 && p.sum > 0.0 ? kind : 0;
    s.p_top = p.top;
    s.p_scale = p.sum > 0.0 ? 1.0 / p.sum : 0.0;
    s.token = -1;
    return s;
}

// Greedy, or nothing has a weight: the first largest logit, or none.
__device__ __forceinline__ int greedy_token(const Total& p, double inv_heat) { return !(inv_heat > 0.0) && p.at != kNowhere ? p.at : -1; }

// `groups` workgroups to a request; each finds its first draft that falls, and its waves take
// the parts of that row.
template <bool F32, bool CAP, int S>
__global__ __launch_bounds__(kWide) void rest_kernel(Args a, Work w, int parts, int groups) {
    constexpr int kWaves = kWide / 64, kHeld = S == 1 ? 8 : 2;  // a row of 262144
    __shared__ U2 table[kSteps];
    __shared__ Total totals[2][kWaves];  // of the rows in hand, and of the drafter's
    __shared__ int falls[kWaves];
    const int tid = (int)threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int r = (int)blockIdx.x / groups, chunk = (int)blockIdx.x - r * groups;
    take_exp2<kWide>(table);
    const Exp exp(table);
    const int start = start_of(a, r), n = start_of(a, r + 1) - start;
    if (chunk == 0) {
        // rows of no request
        if (r == a.requests - 1)
            for (int i = clampi(a.starts[a.requests], 0, a.rows) + tid; i < a.rows; i += kWide) a.out[i] = -1;
        if (r == 0)
            for (int i = tid; i < start; i += kWide) a.out[i] = -1;
    }
    if (n <= 0) {
        if (chunk == 0 && tid == 0) {
            a.accepted[r] = 0;
            w.spots[r] = Spot{};  // pick_kernel reads a row's sums before it looks at the kind
        }
        return;
    }
    const double inv_heat = inv_heat_of(a, r);
    const Part* const own = w.parts + (int64_t)start * parts;
    const Part* const drafts = w.parts + ((int64_t)a.rows + start) * parts;
    const bool drafter = a.draft.x != nullptr;
    __syncthreads();

    // The first draft that falls: a wave to each join, so many rows at a time.
    const int per = drafter ? kWaves / 2 : kWaves;
    int first = n - 1;
    Total p_first{}, q_first{};
    for (int base = 0;; base += per) {
        const int i = base + wave % per;
        const bool of_q = wave >= per;
        // what does not wait for the joins goes out before them
        int token = -1;
        float u = 0.0f, x_at = 0.0f, y_at = 0.0f;
        if (!of_q && i < n - 1) {
            token = a.tokens[start + i + 1];
            u = a.uniforms[2 * (start + i)];
            if (token >= 0 && token < a.vocab) {
                x_at = load1<F32>(a.target, start + i, token);
                if (drafter) y_at = load1<F32>(a.draft, start + i, token);
            } else {
                token = -1;
            }
        }
        if (i < n - of_q) totals[of_q][wave % per] = of_q ? join<CAP, kHeld>(drafts + (int64_t)i * parts, parts, a.draft.cap, inv_heat, exp)
                                                  : join<CAP, kHeld>(own + (int64_t)i * parts, parts, a.target.cap, inv_heat, exp);
        __syncthreads();
        if (!of_q) {
            int fall = kNowhere;
            if (i < n - 1) {
                const bool greedy = !(inv_heat > 0.0);
                const Total p = totals[0][wave], q = totals[1][wave];
                const double p_at = weight_at<CAP>(a.target, token, x_at, p, inv_heat, exp);
                const double q_at = drafter ? weight_at<CAP>(a.draft, token, y_at, q, inv_heat, exp) : 1.0;
                // u q < p, times both sums (a drafter's row without any weight has q = 0)
                const double p_sum = greedy ? 1.0 : p.sum, q_sum = greedy || !drafter || !(q.sum > 0.0) ? 1.0 : q.sum;
                if (!((double)u * q_at * p_sum < p_at * q_sum)) fall = i;
            } else if (i == n - 1) {
                fall = i;  // the last row has no draft
            }
            if (lane == 0) falls[wave] = fall;
        }
        __syncthreads();
        int least = kNowhere;
        for (int j = 0; j < per; ++j) least = falls[j] < least ? falls[j] : least;
        if (least != kNowhere) {
            first = least;
            p_first = totals[0][least - base];
            if (drafter) q_first = totals[1][least - base];
            break;
        }
        __syncthreads();  // the totals are read
    }

    Spot s = spot_of(p_first, start + first, inv_heat, first < n - 1 ? 2 : 1);
    if (s.kind == 2) {
        if (drafter) {
            s.q_top = q_first.top;
            s.q_scale = q_first.sum > 0.0 ? 1.0 / q_first.sum : 0.0;
        } else {
            s.token = a.tokens[s.row + 1];
            if (s.token < 0 || s.token >= a.vocab) s = Spot{s.p_scale, 0.0, s.p_top, 0.0f, s.row, -1, 1, 0};  // nothing to take off p
        }
    }
    if (chunk == 0) {
        if (tid == 0) {
            w.spots[r] = s;
            a.accepted[r] = first;
            if (s.kind == 0) a.out[s.row] = greedy_token(p_first, inv_heat);
        }
        for (int i = tid; i < n; i += kWide)
            if (i != first) a.out[start + i] = i < first ? a.tokens[start + i + 1] : -1;
    }
    if (s.kind != 2) return;  // p's sums are those of its parts

    const Rest<CAP> rest(a, s, inv_heat, exp);
    // Without a drafter's logits only the part that has the token is other than p's (its sum without it is
    // taken anew: a difference would lose what is left).
    const int only = s.token / (512 * S);
    for (int part = drafter ? first_part(chunk, wave) : (chunk == 0 && wave == 0 ? only : parts); part < parts;
         part += drafter ? part_step(groups) : parts) {
        const int begin = part * 512 * S;
        double sum = 0.0;
        if (rest.plain) {
            constexpr int kAtOnce = F32 && S > 2 ? 2 : S;  // four sweeps of both in fp32 are more than 128 registers
#pragma unroll 1
            for (int from = begin; from < begin + 512 * S; from += 512 * kAtOnce) {
                Held<F32, kAtOnce> x, y{};
                x.load(a.target, s.row, from, a.vocab);
                if (drafter) y.load(a.draft, s.row, from, a.vocab);
#pragma unroll
                for (int j = 0; j < kAtOnce; ++j)
#pragma unroll
                    for (int i = 0; i < 8; ++i) sum += rest.template of<true>(from + 512 * j + 8 * lane + i, x.at(j, i), y.at(j, i), exp);
            }
        } else {
            const int end = begin + 512 * S < a.vocab ? begin + 512 * S : a.vocab;
            for (int i = begin + lane; i < end; i += 64)
                sum += rest.template of<false>(i, load1<F32>(a.target, s.row, i), drafter ? load1<F32>(a.draft, s.row, i) : -kInf, exp);
        }
        sum = wave_sum(sum);
        if (lane == 0) w.rest[(int64_t)r * parts + part] = sum;
    }
}

// Inclusive sums over the workgroup's threads, `total` of all; sums: scratch of a value per wave.
__device__ __forceinline__ double group_scan(double v, double* sums, double* total) {
    const int wave = (int)threadIdx.x >> 6;
    v = wave_scan(v);
    __syncthreads();  // the scan before is read
    if ((threadIdx.x & 63) == 63) sums[wave] = v;
    __syncthreads();
    double before = 0.0, all = 0.0;
#pragma unroll
    for (int i = 0; i < kWide / 64; ++i) {
        before += i < wave ? sums[i] : 0.0;
        all += sums[i];
    }
    *total = all;
    return v + before;
}
// The first of the workgroup's threads that is `hit`, the last that has `any`; -1 for none.
struct Ends {
    int first, last;
};
__device__ __forceinline__ Ends group_ends(bool hit, bool any, Ends* ends) {
    const int wave = (int)threadIdx.x >> 6;
    const unsigned long long hits = __ballot(hit), anys = __ballot(any);
    if ((threadIdx.x & 63) == 0)
        ends[wave] = Ends{hits != 0 ? 64 * wave + __ffsll(hits) - 1 : -1, anys != 0 ? 64 * wave + 63 - __clzll(anys) : -1};
    __syncthreads();
    Ends e{-1, -1};
#pragma unroll
    for (int i = 0; i < kWide / 64; ++i) {
        e.first = e.first < 0 ? ends[i].first : e.first;
        e.last = ends[i].last > e.last ? ends[i].last : e.last;
    }
    return e;
}

// DRAFTS: spots and sums are rest_kernel's; else each row is a request and is joined here.
template <bool F32, bool CAP, bool DRAFTS>
__global__ __launch_bounds__(kWide) void pick_kernel(Args a, Work w, Plan plan) {
    __shared__ U2 table[kSteps];
    __shared__ double sums[kWide / 64];
    __shared__ Ends ends[2][kWide / 64];
    __shared__ int ats[kWide / 64];
    __shared__ float tops[kWide / 64];
    __shared__ double before_found;
    const int tid = (int)threadIdx.x, lane = tid & 63, wave = tid >> 6, r = (int)blockIdx.x;
    const int parts = plan.parts;
    Spot s{};
    s.row = r;
    if (DRAFTS) s = w.spots[r];
    const Part* const own = w.parts + (int64_t)s.row * parts;
    const Part none{0.0, -kInf, kNowhere};
    const Part mine = tid < parts ? own[tid] : none;
    const double* const rest = w.rest + (int64_t)r * parts;
    const int size = plan.size(), only = DRAFTS && s.kind == 2 && a.draft.x == nullptr ? s.token / size : -1;
    const bool all_rest = DRAFTS && s.kind == 2 && a.draft.x != nullptr;
    const double my_rest = (all_rest && tid < parts) || tid == only ? rest[tid] : 0.0;
    const double u = (double)(DRAFTS ? a.uniforms[2 * s.row + 1] : a.uniforms[s.row]);
    const double inv_heat = inv_heat_of(a, r);
    take_exp2<kWide>(table);
    const Exp exp(table);
    if constexpr (DRAFTS) {
        if (s.kind == 0) return;
        __syncthreads();
    } else {
        s.kind = 1;
        s.token = -1;
        float top = mine.top;
        for (int i = tid + kWide; i < parts; i += kWide) top = fmaxf(top, own[i].top);
        top = wave_top(top);
        if (lane == 0) tops[wave] = top;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kWide / 64; ++i) top = fmaxf(top, tops[i]);
        s.p_top = top;
        s.p_scale = 1.0;  // weights need not add to one
        if (!(inv_heat > 0.0)) {
            int at = mine.top == top ? mine.at : kNowhere;
            for (int i = tid + kWide; i < parts; i += kWide)
                if (own[i].top == top) at = own[i].at < at ? own[i].at : at;
            at = wave_least(at);
            if (lane == 0) ats[wave] = at;
            __syncthreads();
            if (tid == 0) {
                for (int i = 0; i < kWide / 64; ++i) at = ats[i] < at ? ats[i] : at;
                a.out[r] = at != kNowhere ? at : -1;
            }
            return;
        }
    }

    // The part: the first whose sum with those before it exceeds the goal, else (rounding, or u >= 1)
    // the last with any weight.
    const Scale scale = scale_of<CAP>(s.p_top, a.target.cap, inv_heat, exp);
    const auto part_weight = [&](int i) {
        if (i >= parts) return 0.0;
        if (DRAFTS && s.kind == 2 && (all_rest || i == only)) return i == tid ? my_rest : rest[i];
        const Part p = i == tid ? mine : own[i];
        return p.sum * weight<CAP>(p.top, scale, exp) * s.p_scale;
    };
    double first_weight, upto, total;
    const auto sum_all = [&]() {
        first_weight = part_weight(tid);
        upto = group_scan(first_weight, sums, &total);
        for (int base = kWide; base < parts; base += kWide) {
            double here;
            (void)group_scan(part_weight(base + tid), sums, &here);
            total += here;
        }
    };
    sum_all();
    if (DRAFTS && s.kind == 2 && !(total > 0.0)) {
        s.kind = 1;  // p and q are equal to the last bit
        s.token = -1;
        sum_all();
    }
    const double goal = u * total;
    double before = 0.0, v = first_weight;
    int part = -1, last = -1;
    bool past = true;
    for (int base = 0;;) {
        __syncthreads();  // the round before has read the ends
        const Ends e = group_ends(v > 0.0 && before + upto > goal, v > 0.0, ends[0]);
        if (e.first >= 0) {
            if (tid == e.first) before_found = before + upto - v;
            part = base + e.first;
            past = false;
            break;
        }
        if (e.last >= 0) last = base + e.last;
        base += kWide;
        if (base >= parts) break;
        double here;
        (void)group_scan(v, sums, &here);
        before += here;
        v = part_weight(base + tid);
        upto = group_scan(v, sums, &here);
    }
    __syncthreads();
    if (past) part = last;
    if (part < 0) {  // no weight at all
        if (tid == 0) a.out[s.row] = -1;
        return;
    }

    // The place in it, likewise, by the weights that the part's sum is of.
    const Rest<CAP> of(a, s, inv_heat, exp);
    const bool plain = DRAFTS && s.kind == 2 && (all_rest || part == only) && of.plain;
    const int i0 = part * plan.size() + 2 * tid;
    const bool within = 2 * tid < plan.size();
    double each[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const bool live = within && i0 + i < a.vocab;
        const float x = live ? load1<F32>(a.target, s.row, i0 + i) : -kInf;
        const float y = live && of.minus_q ? load1<F32>(a.draft, s.row, i0 + i) : -kInf;
        each[i] = plain ? of.template of<true>(i0 + i, x, y, exp) : of.template of<false>(i0 + i, x, y, exp);
    }
    const double both = each[0] + each[1], scan = group_scan(both, sums, &total), found = past ? 0.0 : before_found;
    upto = scan + found;
    // of the places before this thread's (0 where none of them has any: then the least weight counts) and its first
    const bool first_hit = !past && each[0] > 0.0 && (scan - both) + found + each[0] > goal;
    const bool hit = first_hit || (!past && each[1] > 0.0 && upto > goal);
    const Ends e = group_ends(hit, each[0] > 0.0 || each[1] > 0.0, ends[1]);
    if (tid == e.first) a.out[s.row] = first_hit ? i0 : i0 + 1;
    if (e.first < 0 && tid == (e.last < 0 ? 0 : e.last)) a.out[s.row] = e.last < 0 ? -1 : (each[1] > 0.0 ? i0 + 1 : i0);
}

int stats_rows(const Args& a) { return a.rows * (a.draft.x != nullptr ? 2 : 1); }
Plan plan_of(const Args& a) { return verify::plan_of(stats_rows(a), a.vocab); }

// A launch counts its threads in 32 bits.
constexpr int64_t kMostThreads = 0xFFFFFFFFll;

size_t part_bytes(const Plan& p) { return (size_t)p.rows * p.parts * sizeof(Part); }
size_t rest_bytes(const Args& a, const Plan& p) {
    return a.starts == nullptr ? 0 : (((size_t)a.requests * p.parts * sizeof(double)) + 15) & ~(size_t)15;
}
size_t spot_bytes(const Args& a) { return a.starts == nullptr ? 0 : (size_t)a.requests * sizeof(Spot); }

template <bool F32, bool CAP, int S>
hipError_t launch_of(const Args& a, const Work& w, const Plan& p, hipStream_t stream) {
    stats_kernel<F32, CAP, S><<<(unsigned)p.groups(), kStatsThreads, 0, stream>>>(a, w, p);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    if (a.starts == nullptr) {
        pick_kernel<F32, CAP, false><<<(unsigned)a.requests, kWide, 0, stream>>>(a, w, p);
        return hipGetLastError();
    }
    const int groups = a.draft.x != nullptr ? rest_groups(a.requests, p.parts) : 1;
    rest_kernel<F32, CAP, S><<<(unsigned)a.requests * (unsigned)groups, kWide, 0, stream>>>(a, w, p.parts, groups);
    e = hipGetLastError();
    if (e != hipSuccess) return e;
    pick_kernel<F32, CAP, true><<<(unsigned)a.requests, kWide, 0, stream>>>(a, w, p);
    return hipGetLastError();
}
template <bool F32, bool CAP>
hipError_t launch_of(const Args& a, const Work& w, const Plan& p, hipStream_t stream) {
    return p.sweeps == 1 ? launch_of<F32, CAP, 1>(a, w, p, stream) : launch_of<F32, CAP, 4>(a, w, p, stream);
}

}  // namespace

bool fits(const Args& a) {
    const Plan p = plan_of(a);
    return p.groups() * kStatsThreads <= kMostThreads && (int64_t)a.requests * rest_groups(a.requests, p.parts) * kWide <= kMostThreads;
}

size_t scratch_bytes(const Args& a) {
    const Plan p = plan_of(a);
    return part_bytes(p) + rest_bytes(a, p) + spot_bytes(a);
}

hipError_t launch(const Args& a, void* scratch, hipStream_t stream) {
    const Plan p = plan_of(a);
    char* at = static_cast<char*>(scratch);
    Work w;
    w.parts = reinterpret_cast<Part*>(at);
    w.rest = reinterpret_cast<double*>(at + part_bytes(p));
    w.spots = reinterpret_cast<Spot*>(at + part_bytes(p) + rest_bytes(a, p));
    const bool cap = a.target.cap > 0.0f || a.draft.cap > 0.0f;
    if (a.target.f32) return cap ? launch_of<true, true>(a, w, p, stream) : launch_of<true, false>(a, w, p, stream);
    return cap ? launch_of<false, true>(a, w, p, stream) : launch_of<false, false>(a, w, p, stream);
}

}  // namespace verify
