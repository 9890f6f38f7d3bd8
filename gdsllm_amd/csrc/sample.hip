// Drawing the next token of each row of logits from a given uniform number.
//
// With m the largest logit and w_i = exp((l_i - m) / T), tokens stand in
// falling order of their logits, equal ones in rising order of their index.  The
// kept tokens are a prefix of that order: the first top_k; of those, every
// token before which less than top_p of their mass lies; of those, the tokens
// with w >= min_p; always the first.  The draw is the first kept token with
//   sum of the kept w up to and with it > u * sum of the kept w.
//
// Nothing is sorted.  fp16 logits have 65536 values, so one pass counts how
// many tokens have each (a histogram of 16-bit counters fills 128 KB of LDS),
// and every cut is found on the counts and on count * w: a prefix of the order
// is a prefix of the values and a number of tokens of one of them.  First the
// binade by its sum, then a value of it to each thread.  fp32 logits take the same
// cuts over three levels of a 32-bit key.  Masses of fp16 rows are 64-bit floating
// sums in a fixed order.  Those of fp32 rows, and of fp16 rows with more than 65535
// equal logits, are 64-bit whole numbers of units of 2^-(62 - L) of the largest
// weight, L = ceil(log2 vocab), so that atomics may add them in any order: each
// weight is off by half a unit at most (less than that: it counts as none), a sum by
// vocab / 2 units, 2^-29 of the largest weight at 131072 tokens, 2^-23 at 2^20.
// Either way a row's token depends on its inputs alone.
//
// A row is one workgroup's, and bound by its latencies: 32000 tokens 15.2 us, of them
// 3.5 to load and count, 4 for the sums of the binades (64-bit arithmetic in all
// waves), 2 for each cut and the draw (two barriers and a chain of 64-bit scans), 1 to
// find the token's index; 64 rows of 128257 on 64 compute units 27 us, 13 of them
// for the two reads of a row.  More registers for the row (8 granules a thread, or 16)
// spill; places looked for by four waves of four values a thread took as long.  fp32
// rows are bound by the 64-bit weight of every token: 32000 tokens 63 to 69 us with
// three cuts, 40 with none, 13 of them for what a row's largest logit alone takes.

#include <algorithm>

#include "common.h"
#include "wave.h"

namespace gdsllm {
namespace {

constexpr int kThreads = 1024;
constexpr int kWaves = kThreads / 64;
constexpr int kMaxVocab = 1 << 20;

struct SampleArgs {
    const void* logits;
    const float *u, *temperature, *top_p, *min_p;
    const int32_t* top_k;
    int64_t* tokens;
    int64_t ld;
    int vocab;
    int shift;  // masses in whole units of 2^-shift: the sum of vocab of them fits 63 bits
};

// 2^y for y <= 0 in 64 bits: the nearest whole number goes to the exponent, the
// rest f (|f| <= 1/2) through sum (f ln 2)^k / k!, k <= 13, whose remainder is
// below 2^-57 of the result.
__device__ __forceinline__ double exp2_neg(double y) {
    y = fmax(y, -1100.0);
    const double n = __builtin_rint(y), f = y - n;
    double p = 1.3691488853904128e-12;   // ln2^13 / 13!, and down
    p = fma(p, f, 2.5678435993488206e-11);
    p = fma(p, f, 4.4455382718708116e-10);
    p = fma(p, f, 7.0549116208011234e-09);
    p = fma(p, f, 1.0178086009239699e-07);
    p = fma(p, f, 1.3215486790144309e-06);
    p = fma(p, f, 1.5252733804059841e-05);
    p = fma(p, f, 1.5403530393381609e-04);
    p = fma(p, f, 1.3333558146428443e-03);
    p = fma(p, f, 9.6181291076284772e-03);
    p = fma(p, f, 5.5504108664821580e-02);
    p = fma(p, f, 2.4022650695910072e-01);
    p = fma(p, f, 6.9314718055994531e-01);
    p = fma(p, f, 1.0);
    return ldexp(p, static_cast<int>(n));
}

struct RowParams {
    double u, c, top_p, min_p;  // c: log2 e / temperature
    int top_k;
    bool greedy;
    __device__ __forceinline__ RowParams(const SampleArgs& a, int row) {
        const float t = a.temperature ? a.temperature[row] : 1.f;
        greedy = !(t > 0.f);
        c = 1.4426950408889634074 / static_cast<double>(t);
        const float uu = a.u[row];
        u = uu > 0.f ? (uu < 1.f ? static_cast<double>(uu) : 1.0) : 0.0;
        top_k = a.top_k ? a.top_k[row] : 0;
        const float p = a.top_p ? a.top_p[row] : 1.f;
        top_p = p < 1.f ? (p > 0.f ? static_cast<double>(p) : 0.0) : 1.0;
        const float mp = a.min_p ? a.min_p[row] : 0.f;
        min_p = mp > 0.f ? static_cast<double>(mp) : 0.0;
    }
    // exp((l - m) / temperature), m the largest logit: 1 at l = m, also where both are infinite.
    __device__ __forceinline__ double weight(float l, float m) const {
        if (m == INFINITY) return l == m ? 1.0 : 0.0;
        return exp2_neg((static_cast<double>(l) - static_cast<double>(m)) * c);
    }
};

typedef unsigned short ushort2_t __attribute__((ext_vector_type(2)));

// Lane l gets lane 63 - l's value.
__device__ __forceinline__ double lane_mirror(double v) { return __shfl_xor(v, 63); }

__device__ __forceinline__ uint32_t rank32(uint32_t b) {
    if (b == 0x80000000u) b = 0;
    return (b & 0x80000000u) ? b : 0x7FFFFFFFu - b;
}
__device__ __forceinline__ bool no_token32(uint32_t b) { return (b & 0x7FFFFFFFu) > 0x7F800000u || b == 0xFF800000u; }
__device__ __forceinline__ float value32(uint32_t rank) {
    return __builtin_bit_cast(float, (rank & 0x80000000u) ? rank : 0x7FFFFFFFu - rank);
}

// The elements of one row, in granules of N aligned elements (8 or 16 bytes).
// Granules that the row fills are loaded whole, the ones at its ends element by
// element.
template <class E, int N_>
struct RowReader {
    static constexpr int N = N_;
    static constexpr int kBytes = N * sizeof(E);
    const E* row;
    int vocab, lead;  // elements of the first granule that lie before the row
    __device__ __forceinline__ RowReader(const E* r, int v) : row(r), vocab(v) {
        lead = static_cast<int>((reinterpret_cast<uintptr_t>(r) & (kBytes - 1)) / sizeof(E));
    }
    __device__ __forceinline__ int granules() const { return (vocab + lead + N - 1) / N; }
    __device__ __forceinline__ int index(int gr) const { return gr * N - lead; }  // of its first element
    // Granule gr of fp16 elements as it lies in memory; past the row: `none`.
    __device__ __forceinline__ uint4 load_packed(int gr, uint32_t none) const {
        const int i0 = index(gr);
        if (i0 >= 0 && i0 + N <= vocab) return *reinterpret_cast<const uint4*>(row + i0);
        uint32_t x[N];
        load(gr, none, x);
        return make_uint4(x[0] | (x[1] << 16), x[2] | (x[3] << 16), x[4] | (x[5] << 16), x[6] | (x[7] << 16));
    }
    // Elements of granule gr; those outside the row get `none`.
    __device__ __forceinline__ void load(int gr, uint32_t none, uint32_t (&x)[N]) const {
        const int i0 = index(gr);
        if (i0 >= 0 && i0 + N <= vocab) {
            uint32_t ws[kBytes / 4];
            if constexpr (kBytes == 16) {
                const uint4 w = *reinterpret_cast<const uint4*>(row + i0);
                ws[0] = w.x, ws[1] = w.y, ws[2] = w.z, ws[3] = w.w;
            } else {
                const uint2 w = *reinterpret_cast<const uint2*>(row + i0);
                ws[0] = w.x, ws[1] = w.y;
            }
#pragma unroll
            for (int j = 0; j < N; ++j)
                x[j] = sizeof(E) == 2 ? (ws[j / 2] >> (16 * (j & 1))) & 0xFFFFu : ws[j % (kBytes / 4)];
        } else {
#pragma unroll
            for (int j = 0; j < N; ++j) x[j] = i0 + j >= 0 && i0 + j < vocab ? row[i0 + j] : none;
        }
    }
};

// Index of element number `which` (from 0, by index) among those for which
// `match` holds.  All threads call it; all get the answer.
template <class R, class F>
__device__ int nth_index(const R& rd, int which, uint32_t none, F match, int* wave_count, int* answer) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int grans = rd.granules();
    const int per = ((grans + kWaves - 1) / kWaves + 63) / 64 * 64, g0 = wave * per, g1 = min(g0 + per, grans);
    int mine = 0;
    for (int gr = g0 + lane; gr < g1; gr += 64) {
        uint32_t x[R::N];
        rd.load(gr, none, x);
#pragma unroll
        for (int j = 0; j < R::N; ++j) mine += match(x[j]) ? 1 : 0;
    }
    mine = wave_sum(mine);
    if (threadIdx.x == 0) *answer = -1;
    if (lane == 0) wave_count[wave] = mine;
    __syncthreads();
    int before = 0;
    for (int w = 0; w < wave; ++w) before += wave_count[w];
    if (which >= before && which < before + mine) {
        int left = which - before;
        for (int gr = g0 + lane; gr - lane < g1; gr += 64) {
            uint32_t x[R::N];
            int c = 0;
            if (gr < g1) {
                rd.load(gr, none, x);
#pragma unroll
                for (int j = 0; j < R::N; ++j) c += match(x[j]) ? 1 : 0;
            }
            const int upto = wave_scan(c);
            if (left >= upto - c && left < upto) {
                int k = left - (upto - c);
#pragma unroll
                for (int j = 0; j < R::N; ++j)
                    if (match(x[j]) && k-- == 0) *answer = rd.index(gr) + j;
            }
            left -= last_lane(upto);
            if (left < 0) break;
        }
    }
    __syncthreads();
    return *answer;
}

// A place in the order: `bin` (a rank), how many tokens of it lie before the
// place, and the number and mass of tokens in the bins before it.
struct Place {
    uint32_t bin;
    int in_bin, count;   // tokens of the bin before the place; tokens before the bin
    double mass, w;      // mass before the bin; weight of the bin's tokens
};

// ---------------------------------------------------------------- 32-bit keys

constexpr int kLevel1 = 4096;  // rank >> 20
constexpr int kLevel2 = 1024;  // (rank >> 10) & 1023; rank & 1023 the third
constexpr int kListed = 12288;

struct Lds32 {
    uint64_t mass1[kLevel1], mass2[kLevel2];
    uint64_t part_mass[kWaves], before_mass, sum;
    uint32_t count1[kLevel1], count2[kLevel2];
    uint32_t list[kListed];  // ranks of the tokens in level-1 bin `listed`
    uint32_t first;
    int part_count[kWaves], before_count, kept, found, answer, counted, length;
};

// One row over 32-bit ranks.  Masses are sums of w in units of 2^-shift, whole
// numbers, so that atomics may add them in any order.  The tokens are counted by
// the upper 12 bits of their rank once; a place is then looked for in its bin
// alone, whose ranks are listed in LDS where they fit.
template <class E>
__device__ void sample_ranks(const SampleArgs& a, int row, Lds32& s) {
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), shift = a.shift;
    const RowReader<E, 4> rd(static_cast<const E*>(a.logits) + row * a.ld, a.vocab);
    const RowParams P(a, row);
    constexpr uint32_t none = sizeof(E) == 2 ? 0xFFFFu : 0xFFFFFFFFu;  // a NaN
    auto bits = [](uint32_t x) { return sizeof(E) == 2 ? __builtin_bit_cast(uint32_t, h2f(x)) : x; };
    auto each = [&](auto f) {
        for (int gr = tid; gr < rd.granules(); gr += kThreads) {
            uint32_t x[4];
            rd.load(gr, none, x);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t b = bits(x[j]);
                if (!no_token32(b)) f(rank32(b));
            }
        }
    };
    if (tid == 0) {
        s.first = 0xFFFFFFFFu;
        s.kept = 0;
        s.counted = 0;
        s.sum = 0;
    }
    for (int i = tid; i < kLevel1; i += kThreads) s.count1[i] = 0, s.mass1[i] = 0;
    for (int i = tid; i < kLevel2; i += kThreads) s.count2[i] = 0, s.mass2[i] = 0;
    __syncthreads();
    uint32_t first = 0xFFFFFFFFu;
    int counted = 0;
    each([&](uint32_t r) {
        first = min(first, r);
        ++counted;
    });
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) first = min(first, static_cast<uint32_t>(__shfl_xor(static_cast<int>(first), o)));
    counted = wave_sum(counted);
    if (lane == 0) {
        atomicMin(&s.first, first);
        atomicAdd(&s.counted, counted);
    }
    __syncthreads();
    first = s.first;
    const int total = s.counted;
    if (total == 0) {
        if (tid == 0) a.tokens[row] = -1;
        return;
    }
    Place at{first, 0, 0, 0.0, 1.0};
    if (!P.greedy) {
        const float top = value32(first);
        const double unit = ldexp(1.0, shift), back = ldexp(1.0, -shift);
        auto add = [&](uint32_t bin, uint32_t r, uint32_t* count, uint64_t* mass) {
            const double w = P.weight(value32(r), top);
            const unsigned long long m = static_cast<unsigned long long>(w * unit + 0.5);
            atomicAdd(&count[bin], 1u);
            atomicAdd(reinterpret_cast<unsigned long long*>(&mass[bin]), m);
            return w;
        };
        int kept = 0;
        each([&](uint32_t r) { kept += add(r >> 20, r, s.count1, s.mass1) >= P.min_p ? 1 : 0; });
        kept = wave_sum(kept);
        if (lane == 0) atomicAdd(&s.kept, kept);
        __syncthreads();
        for (int i = tid; i < kLevel1; i += kThreads)
            if (s.mass1[i]) atomicAdd(reinterpret_cast<unsigned long long*>(&s.sum), static_cast<unsigned long long>(s.mass1[i]));
        __syncthreads();
        int listed = -1;
        // Brings the ranks of level-1 bin `bin` into the list.
        auto list = [&](int bin) {
            if (bin == listed) return;
            listed = bin;
            __syncthreads();
            if (tid == 0) s.length = 0;
            __syncthreads();
            if (s.count1[bin] <= kListed)
                each([&](uint32_t r) {
                    if (static_cast<int>(r >> 20) == bin) s.list[atomicAdd(&s.length, 1)] = r;
                });
            __syncthreads();
        };
        // Counts the tokens whose rank above bit low + 10 is `prefix` by the ten bits from
        // `low` on.  The counters are clear: a search clears what it has read.
        auto fill = [&](int low, uint32_t prefix, int bin) {
            auto one = [&](uint32_t r) {
                if ((r >> (low + 10)) == prefix) add((r >> low) & (kLevel2 - 1), r, s.count2, s.mass2);
            };
            if (s.count1[bin] <= kListed)
                for (int i = tid; i < s.length; i += kThreads) one(s.list[i]);
            else each(one);
            __syncthreads();
        };
        // What lies before this thread's c tokens of mass w, over all threads.
        auto before = [&](int c, uint64_t w, int& ca, uint64_t& wa) {
            const int cu = wave_scan(c);
            const uint64_t wu = wave_scan(w);
            if (lane == 63) {
                s.part_count[wave] = cu;
                s.part_mass[wave] = wu;
            }
            if (tid == 0) {
                s.found = -1;
                s.answer = -1;
            }
            __syncthreads();
            const int own_c = lane < kWaves ? s.part_count[lane] : 0;
            const uint64_t own_w = lane < kWaves ? s.part_mass[lane] : 0;
            const int base_c = wave_scan(own_c) - own_c;
            const uint64_t base_w = wave_scan(own_w) - own_w;
            ca = cu - c + __builtin_amdgcn_readlane(base_c, wave);
            wa = wu - w + __builtin_bit_cast(uint64_t, lane_double(__builtin_bit_cast(double, base_w), wave));
        };
        // The bin in which the place lies, of `per` bins to a thread from bin tid * per on,
        // and what lies before it: n0, m0, of which ca and wa lie before this thread's.
        auto pick = [&](const int* count, const uint64_t* mass, int per, bool by_count, int n, uint64_t m, bool past, int ca,
                        uint64_t wa, int& n0, uint64_t& m0) {
            int last = -1, last_c = 0;  // the place if no bin reaches it: the last that has tokens
            uint64_t last_w = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (i == per) break;
                const int bc = count[i];
                const uint64_t bw = mass[i];
                if (bc > 0) {
                    const bool first = by_count ? ca < n : past ? wa <= m : (wa < m || ca == 0);
                    const bool reached = by_count ? ca + bc >= n : past ? wa + bw > m : wa + bw >= m;
                    if (first && reached && atomicCAS(&s.found, -1, tid * per + i) == -1) {
                        s.before_count = ca;
                        s.before_mass = wa;
                    }
                    last = tid * per + i;
                    last_c = ca;
                    last_w = wa;
                }
                ca += bc;
                wa += bw;
            }
            if (last >= 0 && __ballot(last >= 0) >> lane == 1) atomicMax(&s.answer, last);
            __syncthreads();
            int f = s.found;
            if (f < 0) {
                if (last >= 0 && s.answer == last) {
                    s.before_count = last_c;
                    s.before_mass = last_w;
                }
                f = s.answer;
                __syncthreads();
            }
            n0 = s.before_count;
            m0 = s.before_mass;
            __syncthreads();
            return static_cast<uint32_t>(f);
        };
        auto search2 = [&](bool by_count, int n, uint64_t m, bool past, int& n0, uint64_t& m0, int* tokens) {
            const int c = s.count2[tid];
            const uint64_t w = s.mass2[tid];
            int ca;
            uint64_t wa;
            before(c, w, ca, wa);
            const uint32_t f = pick(&c, &w, 1, by_count, n, m, past, ca + n0, wa + m0, n0, m0);
            if (tokens) *tokens = s.count2[f];
            __syncthreads();
            s.count2[tid] = 0;
            s.mass2[tid] = 0;
            __syncthreads();
            return f;
        };
        // this thread's bins of level 1, which stay
        constexpr int kPer = kLevel1 / kThreads;
        int c1[kPer], before1;
        uint64_t w1[kPer], before1_w;
        {
            int c = 0;
            uint64_t w = 0;
#pragma unroll
            for (int i = 0; i < kPer; ++i) {
                c += c1[i] = s.count1[kPer * tid + i];
                w += w1[i] = s.mass1[kPer * tid + i];
            }
            before(c, w, before1, before1_w);
        }
        __syncthreads();
        auto find = [&](bool by_count, int n, double mass, bool past) {
            const uint64_t m = static_cast<uint64_t>(fmax(mass, 0.0) * unit + (past ? 0.0 : 0.5));
            int n0 = 0, bc = 0;
            uint64_t m0 = 0;
            if (tid == 0) {
                s.found = -1;
                s.answer = -1;
            }
            __syncthreads();
            const uint32_t high = pick(c1, w1, kPer, by_count, n, m, past, before1, before1_w, n0, m0);
            list(high);
            fill(10, high, high);
            const uint32_t bin = (high << 10) | search2(by_count, n, m, past, n0, m0, nullptr);
            fill(0, bin, high);
            const uint32_t low = search2(by_count, n, m, past, n0, m0, &bc);
            Place p;
            p.bin = (bin << 10) | low;
            p.w = P.weight(value32(p.bin), top);
            p.count = n0;
            p.mass = static_cast<double>(m0) * back;
            const double q = p.w > 0.0 ? (fmax(mass, 0.0) - p.mass) / p.w : 0.0;
            if (by_count) p.in_bin = n - n0;
            else p.in_bin = past ? static_cast<int>(fmin(fmax(floor(q), 0.0), bc - 1.0))
                                 : static_cast<int>(fmin(fmax(ceil(q), 1.0), static_cast<double>(bc)));
            return p;
        };
        int cut = total, weighed = total;  // kept tokens; those whose mass `mass` is
        double mass = static_cast<double>(s.sum) * back;
#pragma nounroll
        for (int stage = 0; stage < 5; ++stage) {
            bool by_count = true, past = false;
            int number = 0;
            double amount = 0.0;
            if (stage == 0) {  // the first top_k and their mass
                if (P.top_k <= 0 || P.top_k >= cut) continue;
                number = P.top_k;
            } else if (stage == 1) {  // of those, top_p of their mass
                if (P.top_p >= 1.0) continue;
                by_count = false;
                amount = P.top_p * mass;
            } else if (stage == 2) {  // of those, what min_p keeps; the mass of the kept, where it is not known
                cut = max(min(cut, s.kept), 1);
                if (cut == weighed) continue;
                number = cut;
            } else if (stage == 3) {  // the draw
                by_count = false;
                past = true;
                amount = P.u * mass;
            } else {  // rounding put it behind the last kept token
                if (at.count + at.in_bin < cut) continue;
                number = cut;
            }
            const Place p = find(by_count, number, amount, past);
            if (stage < 3) {
                const int upto = p.count + p.in_bin;
                if (upto <= cut) {
                    weighed = upto;
                    mass = p.mass + p.in_bin * p.w;
                }
                cut = max(min(cut, upto), 1);
            } else {
                at = p;
                at.in_bin -= stage == 4 ? 1 : 0;
            }
        }
    }
    const int i = nth_index(rd, at.in_bin, none,
                            [&](uint32_t x) { return !no_token32(bits(x)) && rank32(bits(x)) == at.bin; },
                            s.part_count, &s.answer);
    if (tid == 0) a.tokens[row] = i;
}

__global__ __launch_bounds__(kThreads) void sample_f32(SampleArgs a) {
    extern __shared__ __attribute__((aligned(16))) char raw[];
    sample_ranks<uint32_t>(a, blockIdx.x, *reinterpret_cast<Lds32*>(raw));
}

// ---------------------------------------------------------------- fp16 logits

// The counters: the values of magnitude h lie in word h, positive ones in its
// low half, negative ones in its high half.  A unit is one binade of one sign,
// 1024 words; in falling order of their values: unit 0 is +inf, 1 .. 31 the
// positive binades, 32 .. 62 the negative ones.
constexpr int kUnits = 63;
constexpr int kMagnitudes = 32768;
constexpr int kListed16 = 2048;  // indices that are sorted by counting

struct Lds16 {
    uint32_t hist[kMagnitudes];
    double mass[64], wave_mass[kWaves];
    Place place;
    int count[64], wave_count[kWaves];
    int top, outside, answer, listed;
};

// Element k (in falling order) of unit u, as fp16 bits.
__device__ __forceinline__ uint32_t unit_bits(int u, int k) {
    const uint32_t base = u == 0 ? 0x7C00u : u < 32 ? static_cast<uint32_t>(31 - u) << 10 : 0x8000u | static_cast<uint32_t>(u - 32) << 10;
    return base | ((u < 32 ? (u == 0 ? 0 : 1023) : 0) ^ (u == 0 ? 0 : k));
}

// One row of fp16 logits by one workgroup.  R > 0: a thread keeps its R granules
// of the row in registers from the count to the search for the token's index; 0:
// they are read twice.
template <int R>
__global__ __launch_bounds__(kThreads) void sample_f16(SampleArgs a) {
    extern __shared__ __attribute__((aligned(16))) char raw[];
    Lds16& s = *reinterpret_cast<Lds16*>(raw);
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), row = blockIdx.x;
    const RowReader<uint16_t, 8> rd(static_cast<const uint16_t*>(a.logits) + row * a.ld, a.vocab);
    constexpr uint32_t none = 0xFFFFu;  // a NaN
    const int grans = rd.granules();

    uint4 keep[R > 0 ? R : 1];
#pragma unroll
    for (int i = 0; i < R; ++i) keep[i] = rd.load_packed(tid + i * kThreads, none);
    for (int i = tid; i < kMagnitudes / 4; i += kThreads) reinterpret_cast<uint4*>(s.hist)[i] = make_uint4(0, 0, 0, 0);
    if (tid == 0) {
        s.top = 0;
        s.outside = 0;
        s.listed = 0;
        s.answer = -1;
    }
    const RowParams P(a, row);
    __syncthreads();

    // -0 becomes +0 by adding +0: equal logits stand together
    auto plain = [](uint32_t two) {
        const half2_t zero = {static_cast<half_t>(0.f), static_cast<half_t>(0.f)};
        return __builtin_bit_cast(uint32_t, __builtin_bit_cast(half2_t, two) + zero);
    };
    half2_t most = {static_cast<half_t>(-INFINITY), static_cast<half_t>(-INFINITY)};
    auto count = [&](const uint4& w) {
        const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t x = plain(ws[j]);
            most = __builtin_elementwise_max(most, __builtin_bit_cast(half2_t, x));
            if (!P.greedy) {
                atomicAdd(&s.hist[x & 0x7FFFu], (x & 0x8000u) ? 0x10000u : 1u);
                atomicAdd(&s.hist[(x >> 16) & 0x7FFFu], (x >> 31) ? 0x10000u : 1u);
            }
        }
    };
    if constexpr (R > 0) {
#pragma unroll
        for (int i = 0; i < R; ++i)
            if (tid + i * kThreads < grans) count(keep[i]);
    } else {
        for (int g0 = tid; g0 < grans; g0 += 4 * kThreads) {
            uint4 w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = rd.load_packed(g0 + i * kThreads, none);
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (g0 + i * kThreads < grans) count(w[i]);
        }
    }
    {
        // the largest logit, as an order-keeping whole number (1023: -inf, so no token)
        const uint32_t x = __builtin_bit_cast(uint32_t, most);
        auto key = [](uint32_t h) { return static_cast<int>((h & 0x8000u) ? 0xFFFFu - h : 0x8000u | h); };
        const int k = wave_max(max(key(x & 0xFFFFu), key(x >> 16)));
        if (lane == 0) atomicMax(&s.top, k);
    }
    __syncthreads();
    const int key = s.top;
    if (key <= 0xFFFF - 0xFC00) {
        if (tid == 0) a.tokens[row] = -1;
        return;
    }
    const uint32_t top_bits = key & 0x8000 ? key & 0x7FFFu : 0xFFFFu - key;
    const float top = h2f(top_bits);
    uint32_t bin = top_bits;
    int which = 0;
    if (!P.greedy) {
        auto counter = [&](uint32_t h) { return static_cast<int>((s.hist[h & 0x7FFFu] >> ((h >> 11) & 16)) & 0xFFFFu); };
        auto weight = [&](uint32_t h) { return h == top_bits ? 1.0 : P.weight(h2f(h), top); };
        auto step_of = [](uint32_t h) {  // between neighbouring values of h's binade
            const uint32_t low = max(h & 0x7C00u, 0x400u);
            return static_cast<double>(h2f(low + 1) - h2f(low));
        };
        // Counts and masses of the units, a wave to the two units of an exponent.  The
        // 1024 values of a binade are evenly spaced, so neighbouring blocks of 64
        // differ by one factor: a lane adds its value of each block by Horner's rule,
        // from the lightest block up, and what is left is the heaviest block's weight
        // times one of 64 that all blocks share.  The largest logit's own block, above
        // which some values lie, is weighed value by value.
        for (int e = wave; e < 32; e += kWaves) {
            const uint32_t first = static_cast<uint32_t>(e) << 10;  // smallest magnitude
            uint32_t n_pos = 0, n_neg = 0;
            double w_pos = 0.0, w_neg = 0.0;
            uint32_t c[16];
#pragma unroll
            for (int j = 0; j < 16; ++j) c[j] = s.hist[first + 64 * j + lane];
            if (e == 31) {  // infinities and NaN: +inf alone of them is a token
                if (lane == 0) {
                    n_pos = c[0] & 0xFFFFu;
                    w_pos = n_pos;
                    c[0] &= 0xFFFF0000u;
                }
                int outside = 0;
#pragma unroll
                for (int j = 0; j < 16; ++j) outside += (c[j] & 0xFFFFu) + (c[j] >> 16);
                outside = wave_sum(outside);
                if (lane == 0 && outside) atomicAdd(&s.outside, outside);
            } else {
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    const ushort2_t two = __builtin_bit_cast(ushort2_t, c[j]);
                    n_pos = __builtin_amdgcn_udot2(two, ushort2_t{1, 0}, n_pos, false);
                    n_neg = __builtin_amdgcn_udot2(two, ushort2_t{0, 1}, n_neg, false);
                }
                if (__any(n_pos + n_neg > 0)) {
                    // blocks behind the heaviest of each sign; the largest logit's own is not among them
                    const int own = e == static_cast<int>((top_bits & 0x7FFFu) >> 10) ? static_cast<int>(top_bits >> 6 & 15) : -1;
                    const bool own_pos = own >= 0 && !(top_bits & 0x8000u), own_neg = own >= 0 && !own_pos;
                    const int jp = own_pos ? own - 1 : 15, jn = own_neg ? own + 1 : 0;
                    const double d = step_of(first) * P.c, up = exp2_neg(-d * (63 - lane)), down = lane_mirror(up);
                    const float heaviest = h2f(lane == 1 ? first + 64 * max(jp, 0) + 63 : 0x8000u | (first + 64 * min(jn, 15)));
                    const double y = lane == 0 ? -64.0 * d : fmin((static_cast<double>(heaviest) - top) * P.c, 0.0);
                    const double f = exp2_neg(lane > 0 && top == INFINITY ? -INFINITY : y);
                    const double r = lane_double(f, 0);
                    if (own < 0) {
#pragma unroll
                        for (int j = 0; j < 16; ++j) {
                            w_pos = fma(w_pos, r, static_cast<double>(c[j] & 0xFFFFu));
                            w_neg = fma(w_neg, r, static_cast<double>(c[15 - j] >> 16));
                        }
                    } else {
#pragma unroll
                        for (int j = 0; j < 16; ++j) {
                            const int k = 15 - j;
                            w_pos = j <= jp ? fma(w_pos, r, static_cast<double>(c[j] & 0xFFFFu)) : w_pos;
                            w_neg = k >= jn ? fma(w_neg, r, static_cast<double>(c[k] >> 16)) : w_neg;
                        }
                    }
                    w_pos *= up * lane_double(f, 1);
                    w_neg *= down * lane_double(f, 2);
                    if (own >= 0) {
                        const uint32_t h = (top_bits & ~63u) + lane;
                        const int n = counter(h);
                        const double w = n ? weight(h) * n : 0.0;
                        w_pos += own_pos ? w : 0.0;
                        w_neg += own_pos ? 0.0 : w;
                    }
                }
            }
            const int all_pos = wave_sum(static_cast<int>(n_pos)), all_neg = wave_sum(static_cast<int>(n_neg));
            w_pos = wave_scan(w_pos);
            w_neg = wave_scan(w_neg);
            if (lane == 63) {
                s.count[31 - e] = all_pos;
                s.mass[31 - e] = w_pos;
                s.count[32 + e] = all_neg;  // [63]: always 0
                s.mass[32 + e] = w_neg;
            }
        }
        __syncthreads();
        // inclusive sums over the units, a unit to a lane, in every wave
        const int unit_n = s.count[lane];
        const double unit_w = s.mass[lane];
        const int upto_n = wave_scan(unit_n);
        const double upto_w = wave_scan(unit_w);
        const int total = last_lane(upto_n);
        if (R == 0 && total + s.outside != grans * 8) {
            // a counter overflowed (over 65535 equal logits): by ranks, 32-bit counters
            __syncthreads();
            sample_ranks<uint16_t>(a, row, *reinterpret_cast<Lds32*>(raw));
            return;
        }
        // The place where the order has had `n` tokens (Count), the first token at
        // which the mass reaches (Reach) or passes (Pass) `m`, or the last token
        // whose weight is at least `m` (Weight).  The unit by its sums, then a value
        // of it to each thread.
        enum Kind { Count, Reach, Pass, Weight };
        auto find = [&](Kind kind, int n, double m) {
            auto at_border = [&](int upto, double mass) {
                return kind == Count ? upto >= n : kind == Pass ? mass > m : mass >= m;
            };
            const uint64_t some = __ballot(unit_n > 0);
            int u;
            if (kind == Weight) {
                // the last unit whose largest value is heavy enough
                const uint64_t heavy = __ballot(unit_n > 0 && weight(unit_bits(lane, 0)) >= m);
                u = heavy ? 63 - __builtin_clzll(heavy) : __builtin_ctzll(some);
            } else {
                const uint64_t hit = __ballot(unit_n > 0 && at_border(upto_n, upto_w));
                u = hit ? __builtin_ctzll(hit) : 63 - __builtin_clzll(some);
            }
            const uint32_t h = unit_bits(u, tid);
            int c = u == 0 && tid > 0 ? 0 : counter(h);
            double w = 0.0;
            if (__any(c > 0)) w = c ? weight(h) : 0.0;
            if (kind == Weight && w < m) c = 0;  // the heavy ones of this unit: their sums are the answer
            int cu = wave_scan(c);
            double wu = wave_scan(w * c);
            if (lane == 63) {
                s.wave_count[wave] = cu;
                s.wave_mass[wave] = wu;
            }
            __syncthreads();
            // the waves' sums, a wave to each of 16 lanes, in every wave
            const int own_n = lane < kWaves ? s.wave_count[lane] : 0;
            const double own_w = lane < kWaves ? s.wave_mass[lane] : 0.0;
            const int waves_n = wave_scan(own_n) + __builtin_amdgcn_readlane(upto_n - unit_n, u);
            const double waves_w = wave_scan(own_w) + lane_double(upto_w - unit_w, u);
            // the one that holds the place (rounding may hide it: then the last with any)
            const uint64_t has = __ballot(own_n > 0), good = __ballot(own_n > 0 && at_border(waves_n, waves_w));
            const int holder = good ? __builtin_ctzll(good) : has ? 63 - __builtin_clzll(has) : 0;
            if (kind == Weight) {
                if (tid == 0) s.place = {0, 0, last_lane(waves_n), lane_double(waves_w, 63), 0.0};
            } else if (wave == holder) {
                cu += __builtin_amdgcn_readlane(waves_n - own_n, holder);
                wu += lane_double(waves_w - own_w, holder);
                const uint64_t in = __ballot(c > 0 && at_border(cu, wu));
                const int l = in ? __builtin_ctzll(in) : 63 - __builtin_clzll(__ballot(c > 0));
                if (lane == l) {
                    Place p{h, 0, cu - c, wu - w * c, w};
                    if (kind == Count) p.in_bin = n - p.count;
                    else if (c == 1 || !in) p.in_bin = kind == Pass ? c - 1 : c;  // hidden: the last token
                    else {
                        const double q = (m - p.mass) / p.w;
                        p.in_bin = kind == Pass ? static_cast<int>(fmin(fmax(floor(q), 0.0), c - 1.0))
                                                : static_cast<int>(fmin(fmax(ceil(q), 1.0), static_cast<double>(c)));
                    }
                    s.place = p;
                }
            }
            __syncthreads();
            return s.place;
        };
        Place at{top_bits, 0, 0, 0.0, 1.0};
        int cut = total, weighed = total;  // kept tokens; those whose mass `mass` is
        double mass = lane_double(upto_w, 63);
#pragma nounroll
        for (int stage = 0; stage < 6; ++stage) {
            Kind kind = Count;
            int number = 0;
            double amount = 0.0;
            if (stage == 0) {  // the first top_k and their mass
                if (P.top_k <= 0 || P.top_k >= cut) continue;
                number = P.top_k;
            } else if (stage == 1) {  // of those, top_p of their mass
                if (P.top_p >= 1.0) continue;
                kind = Reach;
                amount = P.top_p * mass;
            } else if (stage == 2) {  // of those, what min_p keeps
                if (P.min_p <= 0.0) continue;
                kind = Weight;
                amount = P.min_p;
            } else if (stage == 3) {  // the mass of the kept, where no stage found it
                if (cut == weighed) continue;
                number = cut;
            } else if (stage == 4) {  // the draw
                kind = Pass;
                amount = P.u * mass;
            } else {  // rounding put it behind the last kept token
                if (at.count + at.in_bin < cut) continue;
                number = cut;
            }
            const Place p = find(kind, number, amount);
            if (stage < 4) {
                const int upto = p.count + p.in_bin;
                if (upto <= cut) {
                    weighed = upto;
                    mass = p.mass + p.in_bin * p.w;
                }
                cut = max(min(cut, upto), 1);
            } else {
                at = p;
                at.in_bin -= stage == 5 ? 1 : 0;
            }
        }
        bin = at.bin;
        which = at.in_bin;
        __syncthreads();  // the counters have been read: the list takes their place
    }

    // the index of token number `which` of `bin`: its tokens' indices in any order
    // into LDS (over the counters), the one that has `which` before it
    int* list = reinterpret_cast<int*>(s.hist);
    const uint32_t pair = bin | (bin << 16);
    auto look = [&](int gr, const uint4& w) {
        const uint32_t ws[4] = {plain(w.x) ^ pair, plain(w.y) ^ pair, plain(w.z) ^ pair, plain(w.w) ^ pair};
        uint32_t zero = 0;  // a half that is zero borrows from its top bit
#pragma unroll
        for (int j = 0; j < 4; ++j) zero |= (ws[j] - 0x00010001u) & ~ws[j];
        if (!(zero & 0x80008000u)) return;
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (((ws[j / 2] >> (16 * (j & 1))) & 0xFFFFu) == 0) {
                const int n = atomicAdd(&s.listed, 1);
                if (n < kListed16) list[n] = rd.index(gr) + j;
            }
    };
    if constexpr (R > 0) {
#pragma unroll
        for (int i = 0; i < R; ++i)
            if (tid + i * kThreads < grans) look(tid + i * kThreads, keep[i]);
    } else {
        for (int g0 = tid; g0 < grans; g0 += 4 * kThreads) {
            uint4 w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = rd.load_packed(g0 + i * kThreads, none);
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (g0 + i * kThreads < grans) look(g0 + i * kThreads, w[i]);
        }
    }
    __syncthreads();
    const int n = s.listed;
    if (n > kListed16) {
        const int i = nth_index(rd, which, none, [&](uint32_t x) { return (x == 0x8000u ? 0u : x) == bin; }, s.wave_count, &s.answer);
        if (tid == 0) a.tokens[row] = i;
        return;
    }
    for (int i = tid; i < n; i += kThreads) {
        const int mine = list[i];
        int before = 0;
        for (int k = 0; k < n; ++k) before += list[k] < mine ? 1 : 0;
        if (before == which) a.tokens[row] = mine;
    }
}

}  // namespace
}  // namespace gdsllm

using namespace gdsllm;

extern "C" int gdsllm_sample_tokens(const void* logits, int bits, int64_t rows, int64_t vocab, int64_t ld,
                                    const float* u, const float* temperature, const int32_t* top_k, const float* top_p,
                                    const float* min_p, int64_t* tokens, void* stream) {
    const std::string n = "sample_tokens";
    auto bad = [&](const std::string& m) { return set_error(GDSLLM_ERR_INVALID_ARGUMENT, n + ": " + m); };
    if (bits != 16 && bits != 32) return bad("logits must be fp16 or fp32 (bits 16 or 32)");
    if (rows < 0 || rows >= (int64_t(1) << 32) / kThreads) return bad("rows must be in [0, 4194303]");
    if (vocab < 1 || vocab > kMaxVocab) return bad("vocab must be in [1, 1048576], got " + std::to_string(vocab));
    if (rows == 0) return ok();
    if (ld < vocab) return bad("ld < vocab");
    if (!logits || !tokens) return bad("null pointer");
    if (!u) return bad("one uniform number a row expected");
    if (reinterpret_cast<uintptr_t>(logits) % (bits / 8) || reinterpret_cast<uintptr_t>(tokens) % 8 ||
        (reinterpret_cast<uintptr_t>(u) | reinterpret_cast<uintptr_t>(temperature) | reinterpret_cast<uintptr_t>(top_k) |
         reinterpret_cast<uintptr_t>(top_p) | reinterpret_cast<uintptr_t>(min_p)) % 4)
        return bad("misaligned pointer");
    int lg = 0;
    while ((int64_t(1) << lg) < vocab) ++lg;
    const SampleArgs a{logits, u, temperature, top_p, min_p, top_k, tokens, ld, static_cast<int>(vocab), 62 - lg};
    auto launch = [&](auto kernel, size_t lds) {
        if (int rc = prepare_lds(reinterpret_cast<const void*>(kernel), lds)) return rc;
        hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(rows)), dim3(kThreads), lds, as_stream(stream), a);
        return check_hip(hipGetLastError(), "sample_tokens launch");
    };
    static_assert(sizeof(Lds32) <= sizeof(Lds16), "a row that overflows its counters reuses their space");
    const int64_t granules = vocab / 8 + 2;  // at most, wherever the rows begin
    const int rc = bits == 32                 ? launch(&sample_f32, sizeof(Lds32))
                   : granules <= 4 * kThreads ? launch(&sample_f16<4>, sizeof(Lds16))
                                              : launch(&sample_f16<0>, sizeof(Lds16));
    return rc ? rc : ok();
}
