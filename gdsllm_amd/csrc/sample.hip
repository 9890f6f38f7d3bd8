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

struct RowParams {
    double u, t, top_p, min_p;
    int top_k;
    bool greedy;
    __device__ __forceinline__ RowParams(const SampleArgs& a, int row) {
        const float temperature = a.temperature ? a.temperature[row] : 1.f;
        greedy = !(temperature > 0.f);
        t = temperature;
        const float uu = a.u ? a.u[row] : 0.f;
        u = uu > 0.f ? (uu < 1.f ? static_cast<double>(uu) : 1.0) : 0.0;
        top_k = a.top_k ? a.top_k[row] : 0;
        const float p = a.top_p ? a.top_p[row] : 1.f;
        top_p = p < 1.f ? (p > 0.f ? static_cast<double>(p) : 0.0) : 1.0;
        const float mp = a.min_p ? a.min_p[row] : 0.f;
        min_p = mp > 0.f ? static_cast<double>(mp) : 0.0;
    }
    __device__ __forceinline__ double weight(float l, float m) const {
        if (l == m) return 1.0;
        return m == INFINITY ? 0.0 : exp((static_cast<double>(l) - static_cast<double>(m)) / t);
    }
};

// Inclusive sums over a wave.
template <class T>
__device__ __forceinline__ T wave_scan(T v, int lane) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const T u = __shfl_up(v, o);
        if (lane >= o) v += u;
    }
    return v;
}
template <class T>
__device__ __forceinline__ T wave_sum(T v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
    return v;
}

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
            const int upto = wave_scan(c, lane);
            if (left >= upto - c && left < upto) {
                int k = left - (upto - c);
#pragma unroll
                for (int j = 0; j < R::N; ++j)
                    if (match(x[j]) && k-- == 0) *answer = rd.index(gr) + j;
            }
            left -= __shfl(upto, 63);
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
        // counts and masses of the rows of bins, and the tokens that min_p keeps
        int kept = 0;
        for (int r = wave; r < kBinRows; r += kWaves) {
            const int c = bin_count(64 * r + lane);
            double w = 0.0;
            if (__any(c > 0)) {
                if (c > 0) w = P.weight(value16(64 * r + lane), top);
                if (w >= P.min_p) kept += c;
                w *= c;
                w = wave_sum(w);
            }
            const int n = wave_sum(c);
            if (lane == 0) {
                s.mass[r] = w;
                s.count[r] = n;
            }
        }
        kept = wave_sum(kept);
        if (lane == 0) atomicAdd(&s.kept, kept);
        __syncthreads();
        // inclusive sums over the rows, one row a thread
        const int row_n = s.count[tid];
        const double row_w = s.mass[tid];
        int upto_n = wave_scan(row_n, lane);
        double upto_w = wave_scan(row_w, lane);
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
            const int cu = wave_scan(c, lane) + (r > 0 ? s.count[r - 1] : 0);
            const double wu = wave_scan(w * c, lane) + (r > 0 ? s.mass[r - 1] : 0.0);
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
        int n = total;
        double mass = all;
        if (P.top_k > 0 && P.top_k < n) {
            n = P.top_k;
            const Place p = find(true, n, 0.0, false);
            mass = p.mass + p.in_bin * p.w;
        }
        int cut = n;
        if (P.top_p < 1.0) {
            const Place p = find(false, 0, P.top_p * mass, false);
            cut = min(cut, max(p.count + p.in_bin, 1));
        }
        cut = max(min(cut, s.kept), 1);
        if (cut < n) {
            const Place p = find(true, cut, 0.0, false);
            mass = p.mass + p.in_bin * p.w;
        }
        at = find(false, 0, P.u * mass, true);
        if (at.count + at.in_bin >= cut) {
            at = find(true, cut, 0.0, false);
            at.in_bin -= 1;
        }
    }
    const int i = nth_index(rd, at.in_bin, none, [&](uint32_t x) { return !no_token16(x) && rank16(x) == at.bin; },
                            s.part_count, &s.answer);
    if (tid == 0) a.tokens[row] = i;
}

// ---------------------------------------------------------------- 32-bit keys

constexpr int kLevel1 = 4096;  // rank >> 20
constexpr int kLevel2 = 1024;  // (rank >> 10) & 1023; rank & 1023 the third

struct Lds32 {
    uint64_t mass[kLevel1];
    uint32_t count[kLevel1];
    uint64_t part_mass[kWaves];
    int part_count[kWaves];
    int kept, found, answer, counted;
    uint32_t first;
    uint64_t before_mass;
    int before_count;
};

// One row over 32-bit ranks.  Masses are sums of w in units of 2^-shift, whole
// numbers, so that atomics may add them in any order.
template <class E>
__global__ __launch_bounds__(kThreads) void sample_any(SampleArgs a, const int* only_rows, int shift) {
    __shared__ Lds32 s;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, row = blockIdx.x;
    if (only_rows && only_rows[row] == 0) return;
    const RowReader<E, 4> rd(static_cast<const E*>(a.logits) + row * a.ld, a.vocab);
    const RowParams P(a, row);
    constexpr int N = 4;
    constexpr uint32_t none = sizeof(E) == 2 ? 0xFFFFu : 0xFFFFFFFFu;  // a NaN
    auto bits = [](uint32_t x) { return sizeof(E) == 2 ? __builtin_bit_cast(uint32_t, h2f(x)) : x; };
    auto each = [&](auto f) {
        for (int gr = tid; gr < rd.granules(); gr += kThreads) {
            uint32_t x[N];
            rd.load(gr, none, x);
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const uint32_t b = bits(x[j]);
                if (!no_token32(b)) f(rank32(b));
            }
        }
    };
    if (tid == 0) {
        s.first = 0xFFFFFFFFu;
        s.kept = 0;
        s.counted = 0;
    }
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
        auto fixed = [&](uint32_t r) {
            return static_cast<unsigned long long>(P.weight(value32(r), top) * unit + 0.5);
        };
        // Fills the histogram of one level: ranks whose bits above `low + width`
        // equal those of `prefix`.
        auto fill = [&](int low, int bins, uint32_t prefix, bool all_ranks, bool with_mass) {
            __syncthreads();
            for (int i = tid; i < bins; i += kThreads) {
                s.count[i] = 0;
                s.mass[i] = 0;
            }
            __syncthreads();
            each([&](uint32_t r) {
                if (!all_ranks && (r >> (low + 10)) != prefix) return;
                const uint32_t bin = (r >> low) & (bins - 1);
                atomicAdd(&s.count[bin], 1u);
                if (with_mass) atomicAdd(reinterpret_cast<unsigned long long*>(&s.mass[bin]), fixed(r));
            });
            __syncthreads();
        };
        // The bin of this level in which the place lies, and what lies before it
        // (added to n0, m0).  The histogram is left as it was.
        auto search = [&](int bins, bool by_count, int n, uint64_t m, bool past, int& n0, uint64_t& m0) {
            const int per = bins / kThreads > 0 ? bins / kThreads : 1;
            int c = 0;
            uint64_t w = 0;
            const bool on = tid * per < bins;
            if (on)
                for (int i = 0; i < per; ++i) {
                    c += s.count[tid * per + i];
                    w += s.mass[tid * per + i];
                }
            int cu = wave_scan(c, lane);
            uint64_t wu = wave_scan(static_cast<unsigned long long>(w), lane);
            if (lane == 63) {
                s.part_count[wave] = cu;
                s.part_mass[wave] = wu;
            }
            if (tid == 0) s.found = -1;
            __syncthreads();
            for (int v = 0; v < wave; ++v) {
                cu += s.part_count[v];
                wu += s.part_mass[v];
            }
            int ca = n0 + cu - c;
            uint64_t wa = m0 + wu - w;
            int last = -1, last_c = 0;  // the place if no bin reaches it: the last that has tokens
            uint64_t last_w = 0;
            if (on)
                for (int i = 0; i < per; ++i) {
                    const int bc = s.count[tid * per + i];
                    const uint64_t bw = s.mass[tid * per + i];
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
            __syncthreads();
            if (s.found < 0) {
                if (tid == 0) s.answer = -1;
                __syncthreads();
                if (last >= 0) atomicMax(&s.answer, last);
                __syncthreads();
                if (last >= 0 && s.answer == last) {
                    s.found = last;
                    s.before_count = last_c;
                    s.before_mass = last_w;
                }
                __syncthreads();
            }
            const int f = s.found;
            n0 = s.before_count;
            m0 = s.before_mass;
            __syncthreads();
            return static_cast<uint32_t>(f);
        };
        auto find = [&](bool by_count, int n, double mass, bool past) {
            const uint64_t m = static_cast<uint64_t>(fmax(mass, 0.0) * unit + (past ? 0.0 : 0.5));
            int n0 = 0;
            uint64_t m0 = 0;
            fill(20, kLevel1, 0, true, true);
            uint32_t bin = search(kLevel1, by_count, n, m, past, n0, m0);
            fill(10, kLevel2, bin, false, true);
            bin = (bin << 10) | search(kLevel2, by_count, n, m, past, n0, m0);
            fill(0, kLevel2, bin, false, true);
            const uint32_t low = search(kLevel2, by_count, n, m, past, n0, m0);
            const int bc = s.count[low];
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
        // the mass of all tokens, and how many min_p keeps
        int kept = 0;
        unsigned long long sum = 0;
        each([&](uint32_t r) {
            const double w = P.weight(value32(r), top);
            if (w >= P.min_p) ++kept;
            sum += static_cast<unsigned long long>(w * unit + 0.5);
        });
        kept = wave_sum(kept);
        sum = wave_sum(sum);
        if (lane == 0) {
            atomicAdd(&s.kept, kept);
            s.part_mass[wave] = sum;
        }
        __syncthreads();
        uint64_t all = 0;
        for (int w = 0; w < kWaves; ++w) all += s.part_mass[w];
        int n = total;
        double mass = static_cast<double>(all) * back;
        if (P.top_k > 0 && P.top_k < n) {
            n = P.top_k;
            const Place p = find(true, n, 0.0, false);
            mass = p.mass + p.in_bin * p.w;
        }
        int cut = n;
        if (P.top_p < 1.0) {
            const Place p = find(false, 0, P.top_p * mass, false);
            cut = min(cut, max(p.count + p.in_bin, 1));
        }
        cut = max(min(cut, s.kept), 1);
        if (cut < n) {
            const Place p = find(true, cut, 0.0, false);
            mass = p.mass + p.in_bin * p.w;
        }
        at = find(false, 0, P.u * mass, true);
        if (at.count + at.in_bin >= cut) {
            at = find(true, cut, 0.0, false);
            at.in_bin -= 1;
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
        if (over) hipLaunchKernelGGL(sample_any<uint16_t>, grid, block, 0, s, a, static_cast<const int*>(over), shift);
    } else {
        hipLaunchKernelGGL(sample_any<uint32_t>, grid, block, 0, s, a, static_cast<const int*>(nullptr), shift);
    }
    if (int rc = check_hip(hipGetLastError(), "sample_tokens launch")) return rc;
    return ok();
}
