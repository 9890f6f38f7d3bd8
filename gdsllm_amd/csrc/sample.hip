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
// is a prefix of the bins and a number of tokens of one bin.  fp32 logits take
// the same cuts over three levels of a 32-bit key.  All masses are 64-bit
// sums in a fixed order (or integers), so a row's token depends on its inputs
// alone, and a draw next to a border falls on the side where 64 bits put it.

#include <algorithm>

#include "common.h"

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

// Inclusive sums over a wave, in 16-lane rows (DPP shifts) and then across them
// (DPP broadcasts of lanes 15 and 31).
template <int CTRL, int ROWS>
__device__ __forceinline__ int dpp_shift(int v) {
    return __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xF, true);
}
template <int CTRL, int ROWS>
__device__ __forceinline__ uint64_t dpp_shift(uint64_t v) {
    const uint32_t lo = dpp_shift<CTRL, ROWS>(static_cast<int>(v)), hi = dpp_shift<CTRL, ROWS>(static_cast<int>(v >> 32));
    return (static_cast<uint64_t>(hi) << 32) | lo;
}
template <int CTRL, int ROWS>
__device__ __forceinline__ double dpp_shift(double v) {
    return __builtin_bit_cast(double, dpp_shift<CTRL, ROWS>(__builtin_bit_cast(uint64_t, v)));
}
template <class T>
__device__ __forceinline__ T wave_scan(T v) {
    v += dpp_shift<0x111, 0xF>(v);  // row_shr 1, 2, 4, 8
    v += dpp_shift<0x112, 0xF>(v);
    v += dpp_shift<0x114, 0xF>(v);
    v += dpp_shift<0x118, 0xF>(v);
    v += dpp_shift<0x142, 0xA>(v);  // lane 15 of rows 0 and 2 to rows 1 and 3
    v += dpp_shift<0x143, 0xC>(v);  // lane 31 to rows 2 and 3
    return v;
}
// Lane 63's value, in every lane.
__device__ __forceinline__ int last_lane(int v) { return __builtin_amdgcn_readlane(v, 63); }
__device__ __forceinline__ int wave_sum(int v) { return last_lane(wave_scan(v)); }

// Rank of an fp16 value among all of them, 0 for +inf, rising as the value
// falls; +0 and -0 share one.  No token: NaN and -inf.
__device__ __forceinline__ uint32_t rank16(uint32_t h) {
    if (h == 0x8000u) h = 0;
    return (h & 0x8000u) ? h : 0x7FFFu - h;
}
__device__ __forceinline__ bool no_token16(uint32_t h) { return (h & 0x7FFFu) > 0x7C00u || h == 0xFC00u; }
__device__ __forceinline__ float value16(uint32_t rank) { return h2f((rank & 0x8000u) ? rank : 0x7FFFu - rank); }

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

// ---------------------------------------------------------------- fp16 logits

constexpr int kBinRows = 1024;  // 65536 bins as 1024 rows of 64, one lane a bin

struct Lds16 {
    uint32_t hist[32768];  // two 16-bit counters a word
    double mass[kBinRows];
    int count[kBinRows];
    double part_mass[kWaves];
    int part_count[kWaves];
    int first, kept, found_row, answer, counted;
};

__global__ __launch_bounds__(kThreads) void sample_f16(SampleArgs a, int* overflow_rows) {
    extern __shared__ __attribute__((aligned(16))) char raw[];
    Lds16& s = *reinterpret_cast<Lds16*>(raw);
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, row = blockIdx.x;
    const RowReader<uint16_t, 8> rd(static_cast<const uint16_t*>(a.logits) + row * a.ld, a.vocab);
    const RowParams P(a, row);
    constexpr uint32_t none = 0xFFFFu;  // a NaN

    for (int i = tid; i < 32768 / 4; i += kThreads) reinterpret_cast<uint4*>(s.hist)[i] = make_uint4(0, 0, 0, 0);
    if (tid == 0) {
        s.first = 65536;
        s.kept = 0;
        s.counted = 0;
    }
    __syncthreads();
    uint32_t first = 65536;
    int counted = 0;
    for (int gr = tid; gr < rd.granules(); gr += kThreads) {
        uint32_t x[8];
        rd.load(gr, none, x);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            if (no_token16(x[j])) continue;
            const uint32_t r = rank16(x[j]);
            first = min(first, r);
            ++counted;
            if (!P.greedy) atomicAdd(&s.hist[r >> 1], 1u << (16 * (r & 1)));
        }
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) first = min(first, static_cast<uint32_t>(__shfl_xor(static_cast<int>(first), o)));
    counted = wave_sum(counted);
    if (lane == 0) {
        atomicMin(&s.first, static_cast<int>(first));
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
        const float top = value16(first);
        auto bin_count = [&](uint32_t bin) { return static_cast<int>((s.hist[bin >> 1] >> (16 * (bin & 1))) & 0xFFFFu); };
        // Counts and masses of the rows of bins, a row to a thread (each starts at
        // a word of its own, so the threads of a wave read different banks), and the
        // tokens that min_p keeps.
        int kept = 0, row_n = 0;
        double row_w = 0.0;
        for (int i = 0; i < 32; ++i) {
            const int j = (i + tid) & 31;
            const uint32_t two = s.hist[32 * tid + j];
            if (!two) continue;
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const int c = (two >> (16 * k)) & 0xFFFFu;
                if (!c) continue;
                const double w = P.weight(value16(64 * tid + 2 * j + k), top);
                if (w >= P.min_p) kept += c;
                row_n += c;
                row_w = fma(w, static_cast<double>(c), row_w);
            }
        }
        kept = wave_sum(kept);
        if (lane == 0) atomicAdd(&s.kept, kept);
        // inclusive sums over the rows
        int upto_n = wave_scan(row_n);
        double upto_w = wave_scan(row_w);
        if (lane == 63) {
            s.part_count[wave] = upto_n;
            s.part_mass[wave] = upto_w;
        }
        __syncthreads();
        for (int w = 0; w < wave; ++w) {
            upto_n += s.part_count[w];
            upto_w += s.part_mass[w];
        }
        s.count[tid] = upto_n;
        s.mass[tid] = upto_w;
        __syncthreads();
        if (s.count[kBinRows - 1] != total) {
            // a counter overflowed (over 65535 equal logits): the row goes to the other kernel
            if (tid == 0) overflow_rows[row] = 1;
            return;
        }
        const double all = s.mass[kBinRows - 1];
        // The place where the order has had `n` tokens (by_count), or the first
        // token at which the mass reaches `m` (passes it where `past`).
        auto find = [&](bool by_count, int n, double m, bool past) {
            __syncthreads();  // the last search's row has been read
            const double w0 = tid > 0 ? s.mass[tid - 1] : 0.0;
            const int n0 = tid > 0 ? s.count[tid - 1] : 0;
            const int n1 = s.count[tid];
            const double w1 = s.mass[tid];
            if (tid == 0) s.found_row = -1;
            __syncthreads();
            const bool here = by_count ? n0 < n && n <= n1
                                       : (past ? (w0 <= m && w1 > m) : ((w0 < m || n0 == 0) && w1 >= m)) && n1 > n0;
            if (here) atomicMax(&s.found_row, tid);
            __syncthreads();
            int r = s.found_row;
            const bool miss = r < 0;  // rounding hid the border: the last token
            if (miss) {
                r = kBinRows - 1;
                while (r > 0 && s.count[r - 1] == total) --r;
            }
            const int c = bin_count(64 * r + lane);
            const double w = c > 0 ? P.weight(value16(64 * r + lane), top) : 0.0;
            const int cu = wave_scan(c) + (r > 0 ? s.count[r - 1] : 0);
            const double wu = wave_scan(w * c) + (r > 0 ? s.mass[r - 1] : 0.0);
            const bool hit = c > 0 && !miss && (by_count ? cu >= n : past ? wu > m : wu >= m);
            const uint64_t some = __ballot(hit), any = __ballot(c > 0);
            const int l = some ? __builtin_ctzll(some) : 63 - __builtin_clzll(any);
            Place p;
            p.bin = 64 * r + l;
            p.w = __shfl(w, l);
            const int bc = __shfl(c, l);
            p.count = __shfl(cu, l) - bc;
            p.mass = __shfl(wu, l) - p.w * bc;
            if (by_count) p.in_bin = n - p.count;
            else if (!some) p.in_bin = past ? bc - 1 : bc;
            else {
                const double q = (m - p.mass) / p.w;
                p.in_bin = past ? min(max(static_cast<int>(floor(q)), 0), bc - 1) : min(max(static_cast<int>(ceil(q)), 1), bc);
            }
            return p;
        };
        int n = total, cut = total;
        double mass = all;
#pragma nounroll
        for (int stage = 0; stage < 5; ++stage) {
            bool by_count = true, past = false;
            int number = 0;
            double amount = 0.0;
            if (stage == 0) {  // the first top_k and their mass
                if (P.top_k <= 0 || P.top_k >= n) continue;
                number = n = cut = P.top_k;
            } else if (stage == 1) {  // of those, top_p of their mass
                if (P.top_p >= 1.0) continue;
                by_count = false;
                amount = P.top_p * mass;
            } else if (stage == 2) {  // of those, what min_p keeps; the mass of the kept
                cut = max(min(cut, s.kept), 1);
                if (cut == n) continue;
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
            if (stage == 1) {
                cut = min(cut, max(p.count + p.in_bin, 1));
            } else if (stage < 3) {
                mass = p.mass + p.in_bin * p.w;
            } else {
                at = p;
                at.in_bin -= stage == 4 ? 1 : 0;
            }
        }
    }
    const int i = nth_index(rd, at.in_bin, none, [&](uint32_t x) { return !no_token16(x) && rank16(x) == at.bin; },
                            s.part_count, &s.answer);
    if (tid == 0) a.tokens[row] = i;
}

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
__global__ __launch_bounds__(kThreads) void sample_any(SampleArgs a, const int* only_rows, int shift) {
    extern __shared__ __attribute__((aligned(16))) char raw[];
    Lds32& s = *reinterpret_cast<Lds32*>(raw);
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, row = blockIdx.x;
    if (only_rows && only_rows[row] == 0) return;
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
        };
        // Counts the tokens whose rank above bit low + 10 is `prefix` by the ten bits from `low` on.
        auto fill = [&](int low, uint32_t prefix, int bin) {
            __syncthreads();
            for (int i = tid; i < kLevel2; i += kThreads) s.count2[i] = 0, s.mass2[i] = 0;
            __syncthreads();
            auto one = [&](uint32_t r) {
                if ((r >> (low + 10)) == prefix) add((r >> low) & (kLevel2 - 1), r, s.count2, s.mass2);
            };
            if (s.count1[bin] <= kListed)
                for (int i = tid; i < s.length; i += kThreads) one(s.list[i]);
            else each(one);
            __syncthreads();
        };
        // The bin of this level in which the place lies, and what lies before it
        // (added to n0, m0).
        auto search = [&](const uint32_t* count, const uint64_t* mass, int bins, bool by_count, int n, uint64_t m,
                          bool past, int& n0, uint64_t& m0) {
            const int per = bins / kThreads;
            int c = 0;
            uint64_t w = 0;
            for (int i = 0; i < per; ++i) {
                c += count[tid * per + i];
                w += mass[tid * per + i];
            }
            int cu = wave_scan(c);
            uint64_t wu = wave_scan(w);
            if (lane == 63) {
                s.part_count[wave] = cu;
                s.part_mass[wave] = wu;
            }
            if (tid == 0) {
                s.found = -1;
                s.answer = -1;
            }
            __syncthreads();
            for (int v = 0; v < wave; ++v) {
                cu += s.part_count[v];
                wu += s.part_mass[v];
            }
            int ca = n0 + cu - c;
            uint64_t wa = m0 + wu - w;
            int last = -1, last_c = 0;  // the place if no bin reaches it: the last that has tokens
            uint64_t last_w = 0;
            for (int i = 0; i < per; ++i) {
                const int bc = count[tid * per + i];
                const uint64_t bw = mass[tid * per + i];
                if (bc > 0) {
                    const bool before = by_count ? ca < n : past ? wa <= m : (wa < m || ca == 0);
                    const bool reached = by_count ? ca + bc >= n : past ? wa + bw > m : wa + bw >= m;
                    if (before && reached && atomicCAS(&s.found, -1, tid * per + i) == -1) {
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
            if (last >= 0) atomicMax(&s.answer, last);
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
        auto find = [&](bool by_count, int n, double mass, bool past) {
            const uint64_t m = static_cast<uint64_t>(fmax(mass, 0.0) * unit + (past ? 0.0 : 0.5));
            int n0 = 0;
            uint64_t m0 = 0;
            const uint32_t high = search(s.count1, s.mass1, kLevel1, by_count, n, m, past, n0, m0);
            list(high);
            fill(10, high, high);
            const uint32_t bin = (high << 10) | search(s.count2, s.mass2, kLevel2, by_count, n, m, past, n0, m0);
            fill(0, bin, high);
            const uint32_t low = search(s.count2, s.mass2, kLevel2, by_count, n, m, past, n0, m0);
            const int bc = s.count2[low];
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
        int n = total, cut = total;
        double mass = static_cast<double>(s.sum) * back;
#pragma nounroll
        for (int stage = 0; stage < 5; ++stage) {
            bool by_count = true, past = false;
            int number = 0;
            double amount = 0.0;
            if (stage == 0) {  // the first top_k and their mass
                if (P.top_k <= 0 || P.top_k >= n) continue;
                number = n = cut = P.top_k;
            } else if (stage == 1) {  // of those, top_p of their mass
                if (P.top_p >= 1.0) continue;
                by_count = false;
                amount = P.top_p * mass;
            } else if (stage == 2) {  // of those, what min_p keeps; the mass of the kept
                cut = max(min(cut, s.kept), 1);
                if (cut == n) continue;
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
            if (stage == 1) {
                cut = min(cut, max(p.count + p.in_bin, 1));
            } else if (stage < 3) {
                mass = p.mass + p.in_bin * p.w;
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

__global__ void clear_rows(int* rows, int n) {
    const int i = blockIdx.x * blockDim.x + threadIdx.x;
    if (i < n) rows[i] = 0;
}

}  // namespace
}  // namespace gdsllm

using namespace gdsllm;

extern "C" size_t gdsllm_sample_tokens_workspace_size(int64_t rows, int64_t vocab) {
    return rows > 0 && vocab > 65535 ? static_cast<size_t>(rows) * sizeof(int32_t) : 0;
}

extern "C" int gdsllm_sample_tokens(const void* logits, int bits, int64_t rows, int64_t vocab, int64_t ld,
                                    const float* u, const float* temperature, const int32_t* top_k, const float* top_p,
                                    const float* min_p, int64_t* tokens, void* workspace, size_t workspace_bytes,
                                    void* stream) {
    const std::string n = "sample_tokens";
    auto bad = [&](const std::string& m) { return set_error(GDSLLM_ERR_INVALID_ARGUMENT, n + ": " + m); };
    if (bits != 16 && bits != 32) return bad("logits must be fp16 or fp32 (bits 16 or 32)");
    if (rows < 0 || rows > (int64_t(1) << 24)) return bad("bad row count");
    if (vocab < 1 || vocab > kMaxVocab) return bad("vocab must be in [1, 1048576], got " + std::to_string(vocab));
    if (rows == 0) return ok();
    if (ld < vocab) return bad("ld < vocab");
    if (!logits || !tokens) return bad("null pointer");
    if (!u) return bad("one uniform number a row expected");
    if (reinterpret_cast<uintptr_t>(logits) % (bits / 8) || reinterpret_cast<uintptr_t>(tokens) % 8 ||
        (reinterpret_cast<uintptr_t>(u) | reinterpret_cast<uintptr_t>(temperature) | reinterpret_cast<uintptr_t>(top_k) |
         reinterpret_cast<uintptr_t>(top_p) | reinterpret_cast<uintptr_t>(min_p) |
         reinterpret_cast<uintptr_t>(workspace)) % 4)
        return bad("misaligned pointer");
    const SampleArgs a{logits, u, temperature, top_p, min_p, top_k, tokens, ld, static_cast<int>(vocab)};
    const dim3 grid(static_cast<unsigned>(rows)), block(kThreads);
    const hipStream_t s = as_stream(stream);
    int lg = 0;
    while ((int64_t(1) << lg) < vocab) ++lg;
    const int shift = 62 - lg;
    if (bits == 16) {
        const size_t need = gdsllm_sample_tokens_workspace_size(rows, vocab);
        if (need > 0 && (!workspace || workspace_bytes < need))
            return bad("workspace of " + std::to_string(need) + " bytes needed, got " + std::to_string(workspace_bytes));
        int* over = need > 0 ? static_cast<int*>(workspace) : nullptr;
        if (int rc = prepare_lds(reinterpret_cast<const void*>(&sample_f16), sizeof(Lds16))) return rc;
        if (over)
            hipLaunchKernelGGL(clear_rows, dim3(static_cast<unsigned>((rows + 255) / 256)), dim3(256), 0, s, over,
                               static_cast<int>(rows));
        hipLaunchKernelGGL(sample_f16, grid, block, sizeof(Lds16), s, a, over);
        // over 65535 tokens a 16-bit counter can overflow; such rows are left to this
        if (over) {
            if (int rc = prepare_lds(reinterpret_cast<const void*>(&sample_any<uint16_t>), sizeof(Lds32))) return rc;
            hipLaunchKernelGGL(sample_any<uint16_t>, grid, block, sizeof(Lds32), s, a, static_cast<const int*>(over), shift);
        }
    } else {
        if (int rc = prepare_lds(reinterpret_cast<const void*>(&sample_any<uint32_t>), sizeof(Lds32))) return rc;
        hipLaunchKernelGGL(sample_any<uint32_t>, grid, block, sizeof(Lds32), s, a, static_cast<const int*>(nullptr), shift);
    }
    if (int rc = check_hip(hipGetLastError(), "sample_tokens launch")) return rc;
    return ok();
}
