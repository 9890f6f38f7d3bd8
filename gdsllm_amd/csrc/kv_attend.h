// What attention over the 8-bit and the 4-bit cache share: rows and keys of a
// request, the split of the work over workgroups, the join of its parts, the plan
// of a call's launches and the checks of its arguments.  A tile class T (RowTile,
// PromptTile) does a sequence: T::run(args, lds, ...), T::Args, T::Lds, T::kRows,
// T::kD, T::kThreads, T::kPerCu (of them to a compute unit), T::kBegin (blocks that
// the beginning of a sequence counts as) and T::kRowJoin (parts are joined by rows).
#pragma once

#include <algorithm>
#include <climits>

#include "common.h"
#include "wave.h"

namespace gdsllm {
namespace {

typedef float float16_t __attribute__((ext_vector_type(16)));

constexpr float kLog2e = 1.4426950408889634f;
// log2 of a weight where the reference is set, and of the largest that leaves it:
// the lower the reference, the more of a long tail of small weights fp16 holds
// (largest weights of 1 lost tails of 2^-25 a key altogether).  What is left up to
// fp16's 2^16 is for scores so large that fp32 rounds them: PromptTile's exponents
// are off by up to 4 where y is below 2^27, and by 8 below 2^28, where scores are 16
// apart and the reference moves with each.  (Compared as a difference, which fp32
// holds where the sum of the reference and kMost would be rounded.)
constexpr float kSet = 7.f, kMost = 11.f;
constexpr int kSegment = 4096;             // tokens whose block table a workgroup holds in LDS
constexpr int kMaxPages = kSegment / 16;   // segments begin on a block of 64 tokens
constexpr int kBlock = 64;                 // tokens of a unit of work
// Tokens that a request's table may have places for: tiles count them in 32 bits,
// up to a segment past the last one (a sum that wrapped round would be an index).
constexpr int64_t kMostTokens = (int64_t(1) << 31) - 2 * kSegment;

template <class Cache>
struct AttendArgs {
    Cache c;
    const uint16_t* q;
    uint16_t* o;
    const int32_t *tables, *lens, *starts;
    float* part_o;           // [2 * groups][rows of a tile][D]: sums of a sequence's parts
    float2* part_ml;         // [2 * groups][rows of a tile]: maximum and weight sum of each row
    int2* parts;             // [requests][tiles][kv_heads]: first part and their number (0: none)
    int64_t ldq, ldo, ld_table;
    float scale_log2;        // scale * log2 e
    int tokens, requests, q_heads, group, width;
    int min_rows, max_rows;  // requests with other numbers of rows are left to another launch
    int tiles;               // row tiles of a request that the grids have
    int groups;              // workgroups that share the work evenly
    int begin;               // blocks that beginning a sequence counts as
    int zero_other;          // rows of no request are set to zero
};

// A request's rows, in tiles of RT, and the keys they may see.
template <int RT>
struct Rows {
    int start, n, len, rows;
    Rows() = default;
    template <class Args>
    __device__ __forceinline__ Rows(const Args& a, int b) {
        const int s0 = a.starts[b], s1 = a.starts[b + 1], held = a.lens[b];
        start = min(max(s0, 0), a.tokens);
        n = min(max(s1 - start, 0), a.tokens - start);
        len = min(max(held, 0), a.width << a.c.block_log2);
        rows = n * a.group;
        if (rows < a.min_rows || rows > a.max_rows) rows = 0;
    }
    // Keys that the last of rows [r0, r0 + count) sees.
    template <class Args>
    __device__ __forceinline__ int keys(const Args& a, int r0, int count) const {
        const int last = (min(r0 + count, rows) - 1) / a.group;
        return max(len - n + last + 1, 0);
    }
    __device__ __forceinline__ int tiles() const { return (rows + RT - 1) / RT; }
    // Blocks of kBlock tokens to each of its sequences (row tile and kv head).
    __device__ __forceinline__ int blocks() const { return max((len + kBlock - 1) / kBlock, 1); }
    template <class Args>
    __device__ __forceinline__ int work(const Args& a) const { return min(tiles(), a.tiles) * a.c.kv_heads * (blocks() + a.begin); }
};

// f over the values of lanes l % 16 + {0, 16, 32, 48}: every lane gets the result.
template <class F>
__device__ __forceinline__ float over_groups(float v, F f) {
    float a = v, b = v;
    asm volatile("s_nop 1\n\tv_permlane16_swap_b32 %0, %1\n\ts_nop 1" : "+v"(a), "+v"(b));
    v = f(a, b);
    a = v, b = v;
    swap32(a, b);
    return f(a, b);
}

__device__ __forceinline__ float inverse(float l) { return l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l); }

// Rows of no request: before the first one's and behind the last one's.
template <class Args>
__device__ __forceinline__ void zero_other_rows(const Args& a, int D) {
    if (!a.zero_other) return;
    const int before = min(max(a.starts[0], 0), a.tokens), end = min(max(a.starts[a.requests], before), a.tokens);
    for (int64_t i = blockIdx.x; i < before + a.tokens - end; i += gridDim.x) {
        const int64_t t = i < before ? i : end + i - before;
        for (int c = threadIdx.x; c < a.q_heads * D / 8; c += blockDim.x)
            *reinterpret_cast<uint4*>(a.o + t * a.ldo + 8 * c) = make_uint4(0, 0, 0, 0);
    }
}

// One workgroup to a sequence (grid: row tiles times kv heads, requests).  Later
// tiles see more keys: they are dealt first.
template <class T>
__global__ __launch_bounds__(T::kThreads) void attend_whole(typename T::Args a) {
    extern __shared__ __attribute__((aligned(16))) char raw[];
    typename T::Lds& s = *reinterpret_cast<typename T::Lds*>(raw);
    const int b = blockIdx.y, tid = threadIdx.x;
    const int early = T::kThreads < kMaxPages ? -2 : tid < a.width ? a.tables[b * a.ld_table + tid] : -1;
    const Rows<T::kRows> R(a, b);
    const int head = blockIdx.x % a.c.kv_heads;
    for (int tile = a.tiles - 1 - static_cast<int>(blockIdx.x) / a.c.kv_heads; tile < R.tiles(); tile += a.tiles)
        T::run(a, s, b, R, tile, head, 0, R.blocks(), -1, early);
    if (b == 0) zero_other_rows(a, T::kD);
}

// The work as one line of blocks: request after request, in each its row tiles,
// kv heads and blocks of tokens, innermost last; `groups` workgroups take even
// shares of it, so none waits for a long sequence.  Each sums the requests'
// work for itself, a request to a thread a step, and looks up where its share begins.  A sequence
// that lies in several shares leaves a part in each: a workgroup has at most
// two, the one its share begins with and the one it ends in.  A sequence counts
// `begin` blocks more than it has, in front of them: the time it takes to begin one
// (4 us, four loads one after the other), so that no workgroup has several short
// ones beside a full share.

template <class T>
__global__ __launch_bounds__(T::kThreads, T::kPerCu * T::kThreads / 256) void attend_shared(typename T::Args a) {
    constexpr int N = T::kThreads, NW = N / 64;
    extern __shared__ __attribute__((aligned(16))) char raw[];
    typename T::Lds& s = *reinterpret_cast<typename T::Lds*>(raw);
    __shared__ int s_part[NW], s_request, s_begin;
    __shared__ Rows<T::kRows> s_rows;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, wg = blockIdx.x;
    zero_other_rows(a, T::kD);
    int total = 0, share = 0;
    for (int pass = 0; pass < 2; ++pass) {
        int carry = 0;
        for (int b0 = 0; b0 < a.requests; b0 += N) {
            const int b = b0 + tid;
            Rows<T::kRows> R;
            int w = 0;
            if (b < a.requests) {
                R = Rows<T::kRows>(a, b);
                w = R.work(a);
            }
            int upto = wave_scan(w);
            __syncthreads();
            if (lane == 63) s_part[wave] = upto;
            __syncthreads();
            for (int i = 0; i < wave; ++i) upto += s_part[i];
            const int begin = carry + upto - w;
#pragma unroll
            for (int i = 0; i < NW; ++i) carry += s_part[i];
            if (a.requests <= N) {  // one step: the sum is all here
                total = carry;
                share = max((total + a.groups - 1) / a.groups, 4 + a.begin);
            }
            const int at = wg * share;
            if (share > 0 && w > 0 && begin <= at && at < begin + w) s_request = b, s_begin = begin, s_rows = R;
        }
        if (a.requests <= N) break;
        total = carry;
        share = max((total + a.groups - 1) / a.groups, 4 + a.begin);
    }
    __syncthreads();
    auto uniform = [](int v) { return __builtin_amdgcn_readfirstlane(v); };
    share = uniform(share);
    int at = wg * share, b = uniform(s_request), begin = uniform(s_begin);
    const int end = min(at + share, uniform(total));
    if (at >= end) return;
    bool first = true;
    Rows<T::kRows> R;
    R.start = uniform(s_rows.start), R.n = uniform(s_rows.n), R.len = uniform(s_rows.len), R.rows = uniform(s_rows.rows);
    while (at < end) {
        while (at >= begin + R.work(a)) {
            begin += R.work(a);
            R = Rows<T::kRows>(a, ++b);
        }
        const int blocks = R.blocks(), cost = blocks + a.begin, sequence = (at - begin) / cost;
        const int from = at - begin - sequence * cost, to = min(cost, from + end - at);
        const int block0 = max(from - a.begin, 0), block1 = to - a.begin;
        at += to - from;
        if (block1 <= 0) break;  // the share ends before the sequence's first block
        const int head = sequence % a.c.kv_heads, tile = sequence / a.c.kv_heads;
        const bool whole = block0 == 0 && block1 == blocks;
        const int slot = 2 * wg + (first ? 0 : 1);
        if (block0 == 0 && tid == 0)
            a.parts[(static_cast<int64_t>(b) * a.tiles + tile) * a.c.kv_heads + head] =
                make_int2(slot, whole ? 0 : 1 + (blocks - block1 + share - 1) / share);
        T::run(a, s, b, R, tile, head, block0, block1, whole ? -1 : slot, -2);
        if (block0 == 0)  // more rows than the caller said: whole, by whoever begins the tile below
            for (int t = tile + a.tiles; t < R.tiles(); t += a.tiles) T::run(a, s, b, R, t, head, 0, blocks, -1, -2);
        first = false;
    }
}

// Sequences that several workgroups had a part of: one workgroup to a row (to
// every rows-th one where the caller's bound on the rows was too small) adds their
// sums.  Part 0 lies in slot `first`, part i in slot 2 * (first / 2 + i).  Its
// threads first take the parts' maxima and turn them into factors, then D/4
// threads of four channels in each of NG groups run over every NGth part, and the
// groups' sums meet in LDS in a fixed order.
template <class Args, int RT, int D, int THREADS>
__global__ __launch_bounds__(THREADS) void attend_join(Args a, int rows) {
    constexpr int TPR = D / 4, NG = THREADS / TPR, NWV = THREADS / 64, EARLY = THREADS > 256 ? 8 : 2;
    __shared__ float s_f[THREADS], s_m[NWV], s_l[NWV];
    __shared__ __attribute__((aligned(16))) float4_t s_o[THREADS];
    const int b = blockIdx.y, tid = threadIdx.x, wave = tid >> 6;
    const int sequence = blockIdx.x / rows, head = sequence % a.c.kv_heads, row0 = sequence / a.c.kv_heads * RT;
    const int2 d = a.parts[static_cast<int64_t>(b) * a.tiles * a.c.kv_heads + sequence];
    const Rows<RT> R(a, b);
    const int r0 = blockIdx.x % rows, count = min(RT, R.rows - row0);
    if (r0 >= count || d.y == 0) return;  // no such row (d is not set), or whole
    const int parts = d.y;
    for (int r = r0; r < count; r += rows) {
        if (r > r0) __syncthreads();  // the row before has read its sums
        auto at = [&](int i) { return static_cast<int64_t>(i == 0 ? d.x : 2 * (d.x / 2 + i)) * RT + r; };
        auto sums = [&](int i) { return *reinterpret_cast<const float4_t*>(a.part_o + at(i) * D + 4 * (tid % TPR)); };
        // the first parts' sums come in while the factors are made
        float4_t early[EARLY];
#pragma unroll
        for (int k = 0; k < EARLY; ++k) {
            const int i = tid / TPR + k * NG;
            early[k] = i < parts ? sums(i) : float4_t{0.f, 0.f, 0.f, 0.f};
        }
        float my_m = -INFINITY, my_l = 0.f;
        if (tid < parts) {
            const float2 x = a.part_ml[at(tid)];
            my_m = x.x;
            my_l = x.y;
        }
        float m = my_m;
        for (int i = tid + THREADS; i < parts; i += THREADS) m = fmaxf(m, a.part_ml[at(i)].x);
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
        if ((tid & 63) == 0) s_m[wave] = m;
        lds_barrier();
#pragma unroll
        for (int i = 0; i < NWV; ++i) m = fmaxf(m, s_m[i]);
        const float ref = m == -INFINITY ? 0.f : m;
        float l = 0.f;
        float4_t acc = {0.f, 0.f, 0.f, 0.f};
        for (int i0 = 0; i0 < parts; i0 += THREADS) {
            if (i0 > 0) __syncthreads();
            float w = 0.f;
            if (i0 + tid < parts) {
                if (i0 > 0) {
                    const float2 x = a.part_ml[at(i0 + tid)];
                    my_m = x.x;
                    my_l = x.y;
                }
                w = __builtin_amdgcn_exp2f(my_m - ref);
                l = fmaf(my_l, w, l);
            }
            s_f[tid] = w;
            lds_barrier();
            int i = tid / TPR;
            if (i0 == 0) {
#pragma unroll
                for (int k = 0; k < EARLY; ++k, i += NG)
                    if (i < parts) acc += early[k] * s_f[i];
            }
            const int n = min(THREADS, parts - i0);
#pragma unroll 8
            for (; i < n; i += NG) acc += sums(i0 + i) * s_f[i];
        }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) l += __shfl_xor(l, o);
        if ((tid & 63) == 0) s_l[wave] = l;
        s_o[tid] = acc;
        __syncthreads();
        if (tid >= TPR) continue;
        l = 0.f;
#pragma unroll
        for (int i = 0; i < NWV; ++i) l += s_l[i];
#pragma unroll 8
        for (int i = 1; i < NG; ++i) acc += s_o[tid + i * TPR];
        const float inv = inverse(l);
        uint16_t* out = a.o + (R.start + (row0 + r) / a.group) * a.ldo + (head * a.group + (row0 + r) % a.group) * D + 4 * tid;
        uint2 w;
        w.x = pack_h2(static_cast<half_t>(acc[0] * inv), static_cast<half_t>(acc[1] * inv));
        w.y = pack_h2(static_cast<half_t>(acc[2] * inv), static_cast<half_t>(acc[3] * inv));
        *reinterpret_cast<uint2*>(out) = w;
    }
}

// The same where a tile has many rows and a sequence few parts: D/4 threads to a
// row, which go over its parts in order, four of them under way at once.
template <class Args, int RT, int D>
__global__ __launch_bounds__(256) void attend_join_rows(Args a, int blocks) {
    constexpr int TPR = D / 4, RPB = 256 / TPR;
    const int b = blockIdx.y, sequence = blockIdx.x / blocks, head = sequence % a.c.kv_heads, row0 = sequence / a.c.kv_heads * RT;
    const int2 d = a.parts[static_cast<int64_t>(b) * a.tiles * a.c.kv_heads + sequence];
    const Rows<RT> R(a, b);
    const int count = min(RT, R.rows - row0), c = 4 * (threadIdx.x % TPR);
    const int r0 = blockIdx.x % blocks * RPB + threadIdx.x / TPR;
    if (r0 >= count || d.y == 0) return;  // no such row (d is not set where there is none), or whole
    for (int r = r0; r < count; r += blocks * RPB) {
        float m = -INFINITY, l = 0.f;
        float4_t acc = {0.f, 0.f, 0.f, 0.f};
        for (int i0 = 0; i0 < d.y; i0 += 4) {
            float2 ml[4];
            float4_t o[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int i = min(i0 + k, d.y - 1);
                const int64_t at = static_cast<int64_t>(i == 0 ? d.x : 2 * (d.x / 2 + i)) * RT + r;
                ml[k] = a.part_ml[at];
                o[k] = *reinterpret_cast<const float4_t*>(a.part_o + at * D + c);
            }
            float top = m;
#pragma unroll
            for (int k = 0; k < 4; ++k) top = fmaxf(top, ml[k].x);
            const float ref = top == -INFINITY ? 0.f : top, f = __builtin_amdgcn_exp2f(m - ref);
            l *= f;
            acc *= f;
            m = top;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float w = i0 + k < d.y ? __builtin_amdgcn_exp2f(ml[k].x - ref) : 0.f;
                l = fmaf(ml[k].y, w, l);
                acc += o[k] * w;
            }
        }
        const float inv = inverse(l);
        uint16_t* out = a.o + (R.start + (row0 + r) / a.group) * a.ldo + (head * a.group + (row0 + r) % a.group) * D + c;
        uint2 w;
        w.x = pack_h2(static_cast<half_t>(acc[0] * inv), static_cast<half_t>(acc[1] * inv));
        w.y = pack_h2(static_cast<half_t>(acc[2] * inv), static_cast<half_t>(acc[3] * inv));
        *reinterpret_cast<uint2*>(out) = w;
    }
}

// Workgroups of attend_shared that a compute unit holds at once (registers: 16
// rows of accumulators, a tile of codes and Q grow with D).  At D = 256 one, so
// that a long sequence leaves half as many parts: 131072 tokens 36.8 us against
// 41.1 with two.
constexpr int per_cu(int64_t D) { return D == 64 ? 4 : D == 128 ? 3 : 1; }

// One launch of a call: the requests with min_rows to max_rows rows, in tiles of
// `rows` of them.
struct Part {
    bool on = false;
    int rows = 0, min_rows = 0, max_rows = INT_MAX, tiles = 0;
    int64_t sequences = 0;  // (request, row tile, kv head)
    int64_t longest = 0;    // tokens that one may have
    int groups = 0;         // workgroups that share them; 0: one to a sequence
    size_t sums = 0, bytes = 0;
};
struct Plan {
    Part few, many;
    size_t bytes() const { return few.bytes + many.bytes; }
};

constexpr int kCus = 256;  // compute units of the device: the workspace's size goes by it
// Requests of up to kFewRows rows take 16-row tiles, the others 128-row ones, and
// all take 16-row ones, in one launch, where none has more than twice as many (32
// requests of up to 4096 tokens over 8 heads: 8 to 32 rows each 64 us in 16-row
// tiles, 132 with those past 16 in 128-row ones; 16 to 64 rows 111 us in 16-row
// tiles, 146 split at 32; 40 to 128 rows 162 split at 64, 119 in 128-row ones).
constexpr int kFewRows = 32;
// A sequence of up to this many tokens is one workgroup's (4 requests over 8 heads,
// up to 1024 tokens: 12.8 us whole, 17.2 shared out; up to 2048: 20.3 against 17.3).
constexpr int64_t kWholeTokens = 1024;

// Bytes of `groups` workgroups' sums, two parts each of `rows` rows, and of the
// sequences' entries.
size_t part_bytes(int64_t groups, int64_t rows, int64_t sequences, int64_t head_dim) {
    const size_t sums = static_cast<size_t>(groups) * 2 * rows * (head_dim + 2) * sizeof(float);
    return groups ? (sums + sequences * sizeof(int2) + 15) / 16 * 16 : 0;
}

void finish_part(Part* p, int64_t requests, int64_t kv_heads, int64_t head_dim, int64_t max_rows, int64_t max_len,
                 int64_t resident, bool whole) {
    p->on = true;
    p->tiles = static_cast<int>(std::max<int64_t>(1, (max_rows + p->rows - 1) / p->rows));
    p->sequences = requests * kv_heads * p->tiles;
    p->longest = max_len;
    p->groups = whole ? 0 : static_cast<int>(std::min<int64_t>(resident, p->sequences * ((max_len + 255) / 256)));
    p->sums = static_cast<size_t>(p->groups) * 2 * p->rows;
    p->bytes = part_bytes(p->groups, p->rows, p->sequences, head_dim);
}

// Workgroups of 16-row tiles that the device holds at once.
int64_t resident_few(int64_t head_dim) { return per_cu(head_dim) * static_cast<int64_t>(kCus); }

// What the kernels for many rows (prompts) are like: workgroups that a compute
// unit holds at once, and whether work is shared out in 256-row tiles too.
struct Prompts {
    int per_cu;
    bool shares_wide;
};

// One workgroup to a sequence where none is long or there are many of them, else
// as many workgroups as the device holds at once, with even shares.  (256 requests
// of up to 4000 tokens over 8 heads: 218 us whole, 236 shared out; a prompt of 500 tokens
// behind 1500, 128 tiles: 62 whole, 66 shared out; one of 64 in 32 tiles: 57 and 34.)
Plan plan_attend(int64_t requests, int64_t q_heads, int64_t kv_heads, int64_t head_dim, int64_t max_new, int64_t max_len,
                 const Prompts& prompts) {
    Plan p;
    const int64_t rows = max_new * (q_heads / kv_heads);
    const bool many = rows > 2 * kFewRows;
    if (!many || requests > 1) {
        p.few.rows = 16;
        if (many) p.few.max_rows = kFewRows;
        const int64_t most = many ? kFewRows : rows, resident = resident_few(head_dim);
        const int64_t sequences = requests * kv_heads * ((most + 15) / 16);
        finish_part(&p.few, requests, kv_heads, head_dim, most, max_len, resident,
                    max_len <= kWholeTokens || sequences >= (max_len <= 4 * kWholeTokens ? 2 : 8) * resident);
    }
    if (many) {
        const int64_t resident = prompts.per_cu * static_cast<int64_t>(kCus);
        const int64_t sequences = requests * kv_heads * ((rows + 127) / 128), wide_sequences = requests * kv_heads * ((rows + 255) / 256);
        bool wide, whole;
        if (prompts.shares_wide) {
            // 256 rows to a tile (each wave converts half as much) where those are many; whole
            // where two of them come to a compute unit, one after the other: 4 chunks of up
            // to 300 tokens behind up to 5000 take 129 us shared out in 256-row tiles, 160 in
            // 128-row ones and 147 whole, 500 tokens behind 1500 44, 42 and 63
            wide = head_dim <= 128 && 2 * wide_sequences >= resident;
            whole = max_len <= kWholeTokens || (wide ? wide_sequences : sequences) >= 2 * resident;
        } else {
            // 256 rows to a tile where that still leaves two workgroups to a compute unit, one
            // after the other: 4096 tokens of 32 heads over the 8-bit cache 172 us against
            // 188; 4 chunks of 300 tokens 167 against 161
            wide = head_dim <= 128 && wide_sequences >= resident;
            whole = wide || max_len <= (4 * sequences >= resident ? 2 : 1) * kWholeTokens || 2 * sequences >= resident;
        }
        p.many.rows = wide ? 256 : 128;
        if (p.few.on) p.many.min_rows = kFewRows + 1;
        finish_part(&p.many, requests, kv_heads, head_dim, rows, max_len, resident, whole);
    }
    return p;
}

// At least the bytes of plan_attend for every smaller number of requests, max_new
// and max_len too, which need not be less: a prompt of 4096 tokens of 32 heads is
// whole and needs none, 64 tokens behind as many share their work.  Work is
// shared out past kWholeTokens alone, by up to 64 rows of fewer than 8 * resident
// sequences and by 128-row tiles of fewer than resident / 2, or, with
// shares_wide, by tiles of either size of fewer than 2 * resident.
size_t workspace_bound(int64_t requests, int64_t q_heads, int64_t kv_heads, int64_t head_dim, int64_t max_new, int64_t max_len,
                       const Prompts& prompts) {
    if (max_len <= kWholeTokens) return 0;
    const int64_t rows = max_new * (q_heads / kv_heads), units = (max_len + 255) / 256;
    auto part = [&](int64_t tile, int64_t most, int64_t limit, int64_t resident) {
        const int64_t sequences = std::min(requests * kv_heads * std::max<int64_t>(1, (most + tile - 1) / tile), limit);
        return part_bytes(std::min(resident, sequences * units), tile, sequences, head_dim);
    };
    size_t bytes = part(16, std::min<int64_t>(rows, 2 * kFewRows), 8 * resident_few(head_dim), resident_few(head_dim));
    if (rows > 2 * kFewRows) {
        const int64_t resident = prompts.per_cu * static_cast<int64_t>(kCus);
        size_t most = part(128, rows, prompts.shares_wide ? 2 * resident : resident / 2, resident);
        if (prompts.shares_wide && head_dim <= 128) most = std::max(most, part(256, rows, 2 * resident, resident));
        bytes += most;
    }
    return bytes;
}

// Launches one part of a call: W where a workgroup has a whole sequence, S where
// the work is shared out.
template <class W, class S>
int launch_part(typename S::Args a, const Part& p, int64_t blocks, int64_t max_rows, char* workspace, hipStream_t s, const char* where) {
    if (!p.on) return GDSLLM_OK;
    a.min_rows = p.min_rows;
    a.max_rows = p.max_rows;
    a.tiles = p.tiles;
    a.part_o = reinterpret_cast<float*>(workspace);
    a.part_ml = reinterpret_cast<float2*>(a.part_o + p.sums * S::kD);
    a.parts = reinterpret_cast<int2*>(a.part_ml + p.sums);
    a.groups = p.sequences * (blocks + S::kBegin) < (int64_t(1) << 30) ? p.groups : 0;  // the line of blocks is counted in 32 bits
    // (of few long sequences each share begins with one anyway)
    a.begin = 16 * p.sequences >= p.groups ? S::kBegin : 0;
    const unsigned per_request = static_cast<unsigned>(p.tiles) * a.c.kv_heads, requests = a.requests;
    if (a.groups == 0) {
        const size_t lds = sizeof(typename W::Lds);
        if (int rc = prepare_lds(reinterpret_cast<const void*>(&attend_whole<W>), lds)) return rc;
        hipLaunchKernelGGL(attend_whole<W>, dim3(per_request, requests), dim3(W::kThreads), lds, s, a);
        return check_hip(hipGetLastError(), where);
    }
    const size_t lds = sizeof(typename S::Lds);
    if (int rc = prepare_lds(reinterpret_cast<const void*>(&attend_shared<S>), lds)) return rc;
    hipLaunchKernelGGL(attend_shared<S>, dim3(a.groups), dim3(S::kThreads), lds, s, a);
    const int rows = static_cast<int>(std::min<int64_t>(S::kRows, std::max<int64_t>(1, max_rows)));
    if constexpr (S::kRowJoin) {
        constexpr int per = 1024 / S::kD;
        const int n = (rows + per - 1) / per;
        hipLaunchKernelGGL((attend_join_rows<typename S::Args, S::kRows, S::kD>), dim3(per_request * n, requests), dim3(256), 0, s, a, n);
    } else {
        const dim3 join(per_request * rows, requests);
        // few sequences are long, in many parts each
        if (p.sequences * rows <= kCus)
            hipLaunchKernelGGL((attend_join<typename S::Args, S::kRows, S::kD, 1024>), join, dim3(1024), 0, s, a, rows);
        else
            hipLaunchKernelGGL((attend_join<typename S::Args, S::kRows, S::kD, 256>), join, dim3(256), 0, s, a, rows);
    }
    return check_hip(hipGetLastError(), where);
}

bool attend_sizes(int64_t requests, int64_t q_heads, int64_t kv_heads, int64_t head_dim, int64_t max_new, int64_t max_len) {
    return requests >= 0 && requests <= 65535 && kv_heads >= 1 && kv_heads <= 1024 && q_heads >= kv_heads &&
           q_heads <= 16384 && q_heads % kv_heads == 0 && (head_dim == 64 || head_dim == 128 || head_dim == 256) &&
           max_new >= 0 && max_new <= (int64_t(1) << 24) && max_len >= 0 && max_len < (int64_t(1) << 31);
}

// Checks the arguments of a call over `cache` (num_blocks .. head_dim as in
// gdsllm_kv_cache8), fills `a` and plans the launches; *empty: nothing to do.
struct AttendCall {
    Plan plan;
    int64_t blocks = 0, max_rows = 0;
    bool empty = false;
};
template <class Args, class Desc>
int attend_call(const std::string& n, const Desc* cache, const void* q, int64_t ldq, void* o, int64_t ldo, int64_t tokens,
                int64_t q_heads, const int32_t* block_tables, int64_t table_width, int64_t ld_table, const int32_t* lens,
                const int32_t* starts, int64_t requests, float scale, int64_t max_new, int64_t max_len, int zero_other,
                void* workspace, size_t workspace_bytes, const Prompts& prompts, Args& a, AttendCall* call) {
    auto bad = [&](const std::string& m) { return set_error(GDSLLM_ERR_INVALID_ARGUMENT, n + ": " + m); };
    const int64_t D = cache->head_dim;
    if (tokens < 0 || tokens > (int64_t(1) << 30)) return bad("bad token count");
    if (q_heads < 1 || q_heads % cache->kv_heads) return bad("q_heads must be a multiple of kv_heads");
    if (requests < 0 || requests > 65535) return bad("requests must be in [0, 65535]");
    if (table_width < 1 || ld_table < table_width) return bad("ld_table < table_width or an empty table");
    if (table_width > kMostTokens / cache->block_size) return bad("table_width * block_size must be at most 2^31 - 8192");
    if (max_new < 0 || max_len < 0) return bad("negative max_new or max_len");
    if (!(scale > 0.f) || scale > 1e30f) return bad("scale must be positive and finite");
    call->empty = tokens == 0;
    if (call->empty) return GDSLLM_OK;
    if (!q || !o || !starts || (requests > 0 && (!block_tables || !lens))) return bad("null pointer");
    if (ldq < q_heads * D || ldo < q_heads * D) return bad("row stride smaller than a row");
    if (ldq % 8 || ldo % 8) return bad("row strides must be multiples of 8");
    if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(o) | reinterpret_cast<uintptr_t>(workspace)) % 16)
        return bad("q, o and the workspace must be 16-byte aligned");
    if ((reinterpret_cast<uintptr_t>(block_tables) | reinterpret_cast<uintptr_t>(lens) |
         reinterpret_cast<uintptr_t>(starts)) % 4)
        return bad("misaligned pointer");
    if (max_new == 0 || max_new > tokens) max_new = tokens;
    const int64_t most = table_width * cache->block_size;
    if (max_len == 0 || max_len > most) max_len = most;
    if (!attend_sizes(requests, q_heads, cache->kv_heads, D, max_new, max_len)) return bad("sizes out of range");
    if (requests == 0) return bad("no requests for the tokens");
    const Plan& p = call->plan = plan_attend(requests, q_heads, cache->kv_heads, D, max_new, max_len, prompts);
    const size_t need = p.bytes();
    if (need > 0 && (!workspace || workspace_bytes < need))
        return bad("workspace of " + std::to_string(need) + " bytes needed, got " + std::to_string(workspace_bytes));
    a.q = static_cast<const uint16_t*>(q);
    a.o = static_cast<uint16_t*>(o);
    a.tables = block_tables;
    a.lens = lens;
    a.starts = starts;
    a.ldq = ldq;
    a.ldo = ldo;
    a.ld_table = ld_table;
    a.scale_log2 = scale * kLog2e;
    a.tokens = static_cast<int>(tokens);
    a.requests = static_cast<int>(requests);
    a.q_heads = static_cast<int>(q_heads);
    a.group = static_cast<int>(q_heads / cache->kv_heads);
    a.width = static_cast<int>(table_width);
    a.zero_other = zero_other;
    call->max_rows = max_new * a.group;
    if (tokens * q_heads > (int64_t(1) << 30)) return bad("tokens * q_heads must be at most 2^30");
    call->blocks = most / kBlock + 1;
    return GDSLLM_OK;
}

}  // namespace
}  // namespace gdsllm
