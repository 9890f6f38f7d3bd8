// The 4-bit KV cache of a serving loop: the write of a step's keys and values
// (kv4_append) and the rows it holds as fp16 (kv4_values).
//
// Blocks as in the 8-bit cache; codes [block][kv_head][token][head_dim / 2] bytes,
// channel 2i in the low half of byte i, and for each token and group of 32, 64 or
// 128 channels a scale and a bias in fp16, [block][kv_head][group][token], so that
// the tokens of a matrix tile have theirs in one run.  The format is the affine
// one of the 4-bit weights:
//   bias = min x,  scale = fp16((max x - min x) / 15),  code = round((x - bias) / scale),
//   element = fp16(code * scale + bias),
// over the group's finite values.  A token's group depends on that token alone: no
// write rescales another's codes, and the bias, a value of the group, is exact.

#include <algorithm>

#include "kv4_cache.h"
#include "rope.h"

namespace gdsllm {

int kv4_cache_args(const gdsllm_kv_cache4* c, const std::string& where, Kv4Cache* out) {
    auto bad = [&](const std::string& m) { return set_error(GDSLLM_ERR_INVALID_ARGUMENT, where + ": " + m); };
    if (!c) return bad("null cache");
    if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256)
        return bad("head_dim must be 64, 128 or 256, got " + std::to_string(c->head_dim));
    if (c->group_size != 32 && c->group_size != 64 && c->group_size != 128)
        return bad("group_size must be 32, 64 or 128, got " + std::to_string(c->group_size));
    if (c->group_size > c->head_dim) return bad("group_size must not be larger than head_dim");
    if (c->block_size < 16 || c->block_size > 256 || (c->block_size & (c->block_size - 1)))
        return bad("block_size must be 16, 32, 64, 128 or 256, got " + std::to_string(c->block_size));
    if (c->kv_heads < 1 || c->kv_heads > 1024) return bad("kv_heads must be in [1, 1024]");
    if (c->num_blocks < 1 || c->num_blocks > ((int64_t(1) << 31) - 1) / c->block_size)
        return bad("num_blocks must be positive and num_blocks * block_size below 2^31");
    if (c->num_blocks * c->kv_heads >= int64_t(1) << 31) return bad("num_blocks * kv_heads must be below 2^31");
    if (!c->k || !c->v || !c->k_affine || !c->v_affine) return bad("null cache pointer");
    if ((reinterpret_cast<uintptr_t>(c->k) | reinterpret_cast<uintptr_t>(c->v) | reinterpret_cast<uintptr_t>(c->k_affine) |
         reinterpret_cast<uintptr_t>(c->v_affine)) % 16)
        return bad("misaligned cache pointer");
    out->k = static_cast<uint8_t*>(c->k);
    out->v = static_cast<uint8_t*>(c->v);
    out->k_affine = static_cast<uint32_t*>(c->k_affine);
    out->v_affine = static_cast<uint32_t*>(c->v_affine);
    out->num_blocks = static_cast<int>(c->num_blocks);
    out->kv_heads = static_cast<int>(c->kv_heads);
    out->block_log2 = __builtin_ctzll(static_cast<unsigned long long>(c->block_size));
    out->group_log2 = __builtin_ctzll(static_cast<unsigned long long>(c->group_size));
    out->groups = static_cast<int>(c->head_dim / c->group_size);
    return GDSLLM_OK;
}

namespace {

// ----------------------------------------------------------------- kv4_append

struct Append4Args {
    Kv4Cache c;
    const uint16_t *k, *v;
    const int32_t *slots, *positions;
    const float *cos, *sin;
    int64_t ldk, ldv;
    int tokens, half;  // half: pairs of a head that rotate; 0: no rotation
    int max_pos;
    int share;         // waves that share a token's keys (or values)
    int kv_groups;     // workgroups of keys and values; behind them those of q
    RopeRows q;
    int q_units, q_share;
};

// The slot of a row that is written, -1 for padding: a slot outside the
// cache, or a position that the rotation's table does not have.
__device__ __forceinline__ int slot_of(const Append4Args& a, int t) {
    const int s = a.slots[t];
    if (s < 0 || (s >> a.c.block_log2) >= a.c.num_blocks) return -1;
    if (a.half > 0 && static_cast<uint32_t>(a.positions[t]) >= static_cast<uint32_t>(a.max_pos)) return -1;
    return s;
}

// Whether a later row of row t's run of one block has its slot s, by a whole wave.
__device__ __forceinline__ bool written_later(const Append4Args& a, int t, int s, int lane) {
    for (int u0 = t + 1;; u0 += 64) {
        const int u = u0 + lane, v = u < a.tokens ? slot_of(a, u) : -1;
        const uint64_t out = ~__ballot(v >= 0 && (v >> a.c.block_log2) == (s >> a.c.block_log2));
        const int run = out ? __builtin_ctzll(out) : 64;
        if (__ballot(v == s && lane < run)) return true;
        if (run < 64) return false;
    }
}

// f over groups of 1 << LOG2 neighbouring lanes, of 16 at most: every lane gets the result.
template <class F>
__device__ __forceinline__ float over_lanes(float v, int log2, F f) {
    v = f(v, dpp_read<0xB1>(v));
    v = f(v, dpp_read<0x4E>(v));
    if (log2 > 2) v = f(v, dpp_read<0x141>(v));
    if (log2 > 3) v = f(v, dpp_read<0x140>(v));
    return v;
}

// The affine pair (scale, bias) of a group with smallest and largest finite value
// lo and hi (lo > hi: it has none).  The quotient by 15 is one product and its
// remainder's correction: right to the last bit but one, and exact where it has few
// bits, so that its rounding to fp32 is the quotient's (a difference of fp16
// values is a whole number of 2^-24 below 2^41: a fifteenth of it that is no
// middle of two fp32 values is 2^-29 of itself away from one).
__device__ __forceinline__ uint32_t affine_of(float lo, float hi) {
    if (lo > hi) return 0;
    const double span = static_cast<double>(hi) - static_cast<double>(lo);
    double q = span * (1.0 / 15.0);
    q = fma(fma(-q, 15.0, span), 1.0 / 15.0, q);
    uint16_t s = f2h_bits(fp32_rounded(static_cast<float>(q)));
    // the largest element must be finite: 15 * s is exact in fp32, and so is the sum in
    // 64 bits (half a step of s is at most 2^-11 of the span: 64 in all)
    if (hi > 65000.f && 15.0 * static_cast<double>(h2f(s)) + static_cast<double>(lo) >= 65520.0) --s;
    return s | (static_cast<uint32_t>(f2h_bits(lo + 0.f)) << 16);
}

// A dword of codes round((x - bias) / scale), ties to even, in [0, 15], of eight
// values.  NaN and what lies below is 0, and all are where the scale is 0.  A
// candidate in fp32 whose remainder, off by at most 2^-24 (|x - bias| + scale / 2) <
// 2^-19 scale, is less than half a scale by more than that is the code (a group's
// x - bias is at most 22 scales, where the scale rounds 22/15 steps of 2^-24 to one).
// Where that does not decide, the remainder in 64 bits, which is exact, does.
__device__ __forceinline__ uint32_t codes_of(const float (&x)[8], float scale, float bias) {
    const float inv = scale > 0.f ? 1.f / scale : 0.f, sure = scale * 0.49998f;
    float n[8];
    bool all_sure = true;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const float d = x[j] - bias;
        n[j] = __builtin_rintf(d * inv);
        all_sure &= fabsf(fmaf(-n[j], scale, d)) < sure;
    }
    if (!all_sure && scale > 0.f) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            if (!(fabsf(x[j]) < INFINITY)) continue;
            const double d = static_cast<double>(x[j]) - static_cast<double>(bias), s = scale;
            const double r2 = 2.0 * fma(-static_cast<double>(n[j]), s, d);
            const bool odd = static_cast<int>(n[j]) & 1;
            if (r2 > s || (r2 == s && odd)) n[j] += 1.f;
            else if (r2 < -s || (r2 == -s && odd)) n[j] -= 1.f;
        }
    }
    uint32_t w = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) w |= static_cast<uint32_t>(fminf(fmaxf(n[j], 0.f), 15.f)) << (4 * j);
    return w;
}

// Keys or values of one token, `share` waves to it, 64 / C heads to a wave at a
// time and a chunk of eight channels to a lane.  2000 tokens of 32 heads of 128
// channels, with as many of q: 20.6 us (26.9 with every quotient and remainder in
// 64 bits), 3.7 TB/s; 17.6 without the writes.
template <int D, bool NEIGHBOURS>
__device__ void append4_rows(const Append4Args& a, int wave) {
    constexpr int C = D / 8, HEADS = 64 / C;
    const int lane = threadIdx.x & 63, ch = lane % C;
    const int t = wave / (2 * a.share), kind = wave / a.share & 1, part = wave % a.share;
    if (t >= a.tokens) return;
    const int s = slot_of(a, t);
    if (s < 0 || written_later(a, t, s, lane)) return;
    const int bs = 1 << a.c.block_log2, page = s >> a.c.block_log2, off = s & (bs - 1);
    const bool is_k = kind == 0;
    const uint16_t* row = is_k ? a.k + t * a.ldk : a.v + t * a.ldv;
    uint8_t* codes = is_k ? a.c.k : a.c.v;
    uint32_t* affine = is_k ? a.c.k_affine : a.c.v_affine;
    const int hc = NEIGHBOURS ? a.half >> 2 : a.half >> 3;  // chunks that hold all pairs, or the first halves
    const bool turns = is_k && ch < (NEIGHBOURS ? hc : 2 * hc), first = ch < hc;
    const float *cs = nullptr, *sn = nullptr;
    if (turns) {
        const int64_t at = static_cast<int64_t>(a.positions[t]) * a.half + (NEIGHBOURS ? 4 * ch : 8 * (first ? ch : ch - hc));
        cs = a.cos + at;
        sn = a.sin + at;
    }
    const int lanes_log2 = a.c.group_log2 - 3, group = ch >> lanes_log2;
    for (int head = part * HEADS + lane / C; head < a.c.kv_heads; head += a.share * HEADS) {
        const uint16_t* p = row + head * D;
        uint4 x = *reinterpret_cast<const uint4*>(p + 8 * ch);
        if (turns) {
            if constexpr (NEIGHBOURS) {
                Angles<4> g;
                g.load(cs, sn);
                x = turn_neighbours(x, g);
            } else {
                const uint4 other = *reinterpret_cast<const uint4*>(p + 8 * (first ? ch + hc : ch - hc));
                Angles<8> g;
                g.load(cs, sn);
                x = turn_half(x, other, first, g);
            }
        }
        float f[8], lo = INFINITY, hi = -INFINITY;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            f[j] = h2f(half_of(x, j));
            lo = fminf(lo, f[j]);
            hi = fmaxf(hi, f[j]);
        }
        if (!(lo > -INFINITY && hi < INFINITY)) {  // of the finite ones
            lo = INFINITY, hi = -INFINITY;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const bool finite = fabsf(f[j]) < INFINITY;
                lo = fminf(lo, finite ? f[j] : INFINITY);
                hi = fmaxf(hi, finite ? f[j] : -INFINITY);
            }
        }
        lo = over_lanes(lo, lanes_log2, [](float u, float v) { return fminf(u, v); });
        hi = over_lanes(hi, lanes_log2, [](float u, float v) { return fmaxf(u, v); });
        const uint32_t ab = affine_of(lo, hi);
        const uint32_t w = codes_of(f, h2f(ab & 0xFFFFu), h2f(ab >> 16));
        const int64_t base = static_cast<int64_t>(page) * a.c.kv_heads + head;
        *reinterpret_cast<uint32_t*>(codes + ((base << a.c.block_log2) + off) * (D / 2) + 4 * ch) = w;
        if ((ch & ((1 << lanes_log2) - 1)) == 0) affine[((base * a.c.groups + group) << a.c.block_log2) + off] = ab;
    }
}

// Workgroups [0, kv_groups): keys and values; behind them q, four heads to a
// thread, as in rope.  8192 tokens of 32 heads of 256 channels over two: 69 us, of
// which q's 268 MB take 57 at 4.7 TB/s.
template <int D, bool NEIGHBOURS>
__global__ __launch_bounds__(256) void kv4_append(Append4Args a) {
    if (static_cast<int>(blockIdx.x) < a.kv_groups) {
        append4_rows<D, NEIGHBOURS>(a, static_cast<int>(blockIdx.x) * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6));
        return;
    }
    const int per = 256 / a.q_units, g = threadIdx.x / a.q_units;
    if (g >= per) return;
    const int64_t group = static_cast<int64_t>(blockIdx.x - a.kv_groups) * per + g, t = group / a.q_share;
    if (t >= a.tokens) return;
    const bool live = slot_of(a, static_cast<int>(t)) >= 0;
    const int64_t at = live ? static_cast<int64_t>(a.positions[t]) * a.half : 0;
    rope_unit<NEIGHBOURS, 4>(a.q, D, a.half, t, threadIdx.x - g * a.q_units, static_cast<int>(group - t * a.q_share), a.q_share, live,
                             a.cos + at, a.sin + at);
}

// ----------------------------------------------------------------- kv4_values

struct Values4Args {
    Kv4Cache c;
    const int32_t* slots;
    uint16_t *k, *v;
    int64_t rows;
};

// 256 / C rows of one head to a workgroup, a chunk of eight channels to a thread:
// neighbouring rows' codes and affine pairs lie side by side where they are neighbouring
// tokens.  Bound by the bytes, most of them the rows': 8192 rows of 32 heads of 128
// channels 26 us, 6.7 TB/s (stores that stay in the caches 38; a row's heads to a
// workgroup, half a cache line of each head's codes, 55).
template <int D>
__global__ __launch_bounds__(256) void kv4_values(Values4Args a) {
    constexpr int C = D / 8;
    const NibUnpack nib;
    const int head = blockIdx.x % a.c.kv_heads, ch = threadIdx.x % C;
    const int64_t row = static_cast<int64_t>(blockIdx.x / a.c.kv_heads) * (256 / C) + threadIdx.x / C;
    if (row >= a.rows) return;
    const int s = a.slots[row], page = s >> a.c.block_log2;
    uint4 k = make_uint4(0, 0, 0, 0), v = k;
    if (s >= 0 && page < a.c.num_blocks) {
        const int off = s & ((1 << a.c.block_log2) - 1), group = ch >> (a.c.group_log2 - 3);
        const int64_t base = static_cast<int64_t>(page) * a.c.kv_heads + head;
        const int64_t code = ((base << a.c.block_log2) + off) * (D / 2) + 4 * ch;
        const int64_t pair = ((base * a.c.groups + group) << a.c.block_log2) + off;
        const uint32_t wk = *reinterpret_cast<const uint32_t*>(a.c.k + code), wv = *reinterpret_cast<const uint32_t*>(a.c.v + code);
        const uint32_t ak = a.c.k_affine[pair], av = a.c.v_affine[pair];
        k = rising_from_pairs(elements8(nib, wk, ak));
        v = rising_from_pairs(elements8(nib, wv, av));
    }
    const int64_t to = ((row * a.c.kv_heads + head) * C + ch) * 8;
    store_nt16(a.k + to, k);
    store_nt16(a.v + to, v);
}

}  // namespace
}  // namespace gdsllm

using namespace gdsllm;

extern "C" int gdsllm_kv4_append(const gdsllm_kv_cache4* cache, const void* k, int64_t ldk, const void* v, int64_t ldv,
                                 const int32_t* slots, int64_t tokens, const void* q, int64_t ldq, void* q_out,
                                 int64_t q_heads, const int32_t* positions, const float* cos, const float* sin,
                                 int64_t rotary, int64_t max_pos, int neighbours, void* stream) {
    const std::string n = "kv4_append";
    auto bad = [&](const std::string& m) { return set_error(GDSLLM_ERR_INVALID_ARGUMENT, n + ": " + m); };
    Append4Args a{};
    if (int rc = kv4_cache_args(cache, n, &a.c)) return rc;
    const int64_t D = cache->head_dim;
    if (tokens < 0 || tokens > (int64_t(1) << 30)) return bad("bad token count");
    if (rotary < 0 || rotary > D || rotary % 16)
        return bad("rotary must be a multiple of 16 in [0, head_dim], got " + std::to_string(rotary));
    if (q && !rotary) return bad("q is given without a rotation");
    if (q && (q_heads < 1 || q_heads > 16384)) return bad("q_heads must be in [1, 16384]");
    if (tokens == 0) return ok();
    if (!k || !v || !slots || (q && !q_out)) return bad("null pointer");
    if (rotary && (!positions || !cos || !sin)) return bad("a rotation needs positions, cos and sin");
    if (rotary && (max_pos < 1 || max_pos > (int64_t(1) << 31) - 1)) return bad("bad number of positions");
    if (ldk < cache->kv_heads * D || ldv < cache->kv_heads * D || (q && ldq < q_heads * D))
        return bad("row stride smaller than a row");
    if (ldk % 8 || ldv % 8 || (q && ldq % 8)) return bad("row strides must be multiples of 8");
    if ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) | reinterpret_cast<uintptr_t>(q) |
         reinterpret_cast<uintptr_t>(q_out)) % 16)
        return bad("k, v, q and q_out must be 16-byte aligned");
    if ((reinterpret_cast<uintptr_t>(slots) | reinterpret_cast<uintptr_t>(positions)) % 4 ||
        (reinterpret_cast<uintptr_t>(cos) | reinterpret_cast<uintptr_t>(sin)) % 16)
        return bad("misaligned pointer (cos and sin: 16 bytes)");
    if (q && q == q_out) return bad("q_out must not be q");
    a.k = static_cast<const uint16_t*>(k);
    a.v = static_cast<const uint16_t*>(v);
    a.slots = slots;
    a.positions = positions;
    a.cos = cos;
    a.sin = sin;
    a.ldk = ldk;
    a.ldv = ldv;
    a.tokens = static_cast<int>(tokens);
    a.half = static_cast<int>(rotary / 2);
    a.max_pos = static_cast<int>(max_pos);
    // waves of a token's keys: one for each 64 chunks while tokens are few, fewer for a prompt
    const int64_t most = (cache->kv_heads * D / 8 + 63) / 64;
    a.share = static_cast<int>(std::min<int64_t>(most, std::max<int64_t>(1, 32 * static_cast<int64_t>(cu_count()) / (2 * tokens))));
    const int64_t kv_groups = (tokens * 2 * a.share + 3) / 4;
    int64_t q_groups = 0;
    if (q) {
        a.q = {static_cast<const uint16_t*>(q), nullptr, static_cast<uint16_t*>(q_out), nullptr, ldq, 0, q_heads * D, 0,
               static_cast<int>(q_heads), static_cast<int>(q_heads)};
        a.q_units = rope_units(static_cast<int>(D), a.half, neighbours != 0);
        a.q_share = static_cast<int>((q_heads + 3) / 4);
        const int per = 256 / a.q_units;
        q_groups = (tokens * a.q_share + per - 1) / per;
    }
    if ((kv_groups + q_groups) * 256 >= (int64_t(1) << 32) || tokens * 2 * a.share >= (int64_t(1) << 31))
        return bad("too many tokens and heads for one call");
    a.kv_groups = static_cast<int>(kv_groups);
    const dim3 grid(static_cast<unsigned>(kv_groups + q_groups));
    const hipStream_t s = as_stream(stream);
#define GDSLLM_APPEND4(DIM)                                                                             \
    if (D == DIM) {                                                                                     \
        if (neighbours) hipLaunchKernelGGL((kv4_append<DIM, true>), grid, dim3(256), 0, s, a);          \
        else hipLaunchKernelGGL((kv4_append<DIM, false>), grid, dim3(256), 0, s, a);                    \
    }
    GDSLLM_APPEND4(64)
    GDSLLM_APPEND4(128)
    GDSLLM_APPEND4(256)
#undef GDSLLM_APPEND4
    if (int rc = check_hip(hipGetLastError(), "kv4_append launch")) return rc;
    return ok();
}

extern "C" int gdsllm_kv4_values(const gdsllm_kv_cache4* cache, const int32_t* slots, int64_t rows, void* k, void* v,
                                 void* stream) {
    const std::string n = "kv4_values";
    auto bad = [&](const std::string& m) { return set_error(GDSLLM_ERR_INVALID_ARGUMENT, n + ": " + m); };
    Values4Args a{};
    if (int rc = kv4_cache_args(cache, n, &a.c)) return rc;
    if (rows < 0 || rows > (int64_t(1) << 30)) return bad("bad row count");
    if (rows == 0) return ok();
    if (!slots || !k || !v) return bad("null pointer");
    if (reinterpret_cast<uintptr_t>(slots) % 4 || (reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) % 16)
        return bad("misaligned pointer (k and v: 16 bytes)");
    a.slots = slots;
    a.k = static_cast<uint16_t*>(k);
    a.v = static_cast<uint16_t*>(v);
    a.rows = rows;
    const int64_t D = cache->head_dim, per = 256 / (D / 8), grid = (rows + per - 1) / per * cache->kv_heads;
    if (grid * 256 >= (int64_t(1) << 32)) return bad("too many rows and heads for one call");
    const dim3 g(static_cast<unsigned>(grid));
    const hipStream_t s = as_stream(stream);
    if (D == 64) hipLaunchKernelGGL(kv4_values<64>, g, dim3(256), 0, s, a);
    else if (D == 128) hipLaunchKernelGGL(kv4_values<128>, g, dim3(256), 0, s, a);
    else hipLaunchKernelGGL(kv4_values<256>, g, dim3(256), 0, s, a);
    if (int rc = check_hip(hipGetLastError(), "kv4_values launch")) return rc;
    return ok();
}
