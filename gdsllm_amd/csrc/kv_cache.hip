// The 8-bit KV cache of a serving loop: which blocks each request holds
// (kv_assign) and the write of a step's keys and values into them (kv_append).
//
// A layer's cache is a pool of blocks of `block_size` tokens.  Codes lie as
// [block][kv_head][token][head_dim], so that one head's block is one
// contiguous run, and each (block, head) has one fp32 scale for its keys and
// one for its values: element = scale * code.
//
// The scales this file writes are powers of two.  x / scale and scale / scale
// are then exact, each code is one rounding of the fp16 value, and when a later
// token makes a block's scale grow the old codes are rescaled exactly in e4m3
// (but for codes that become subnormal) and with one more rounding in int8.
// That costs at most one bit of the range and makes results independent of the
// order of the arithmetic.

#include <algorithm>

#include "kv_cache.h"
#include "wave.h"

namespace gdsllm {

int kv_cache_args(const gdsllm_kv_cache8* c, const std::string& where, KvCache* out) {
    auto bad = [&](const std::string& m) { return set_error(GDSLLM_ERR_INVALID_ARGUMENT, where + ": " + m); };
    if (!c) return bad("null cache");
    if (c->format != GDSLLM_KV_E4M3 && c->format != GDSLLM_KV_INT8) return bad("unknown cache format");
    if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256)
        return bad("head_dim must be 64, 128 or 256, got " + std::to_string(c->head_dim));
    if (c->block_size < 16 || c->block_size > 256 || (c->block_size & (c->block_size - 1)))
        return bad("block_size must be 16, 32, 64, 128 or 256, got " + std::to_string(c->block_size));
    if (c->kv_heads < 1 || c->kv_heads > 1024) return bad("kv_heads must be in [1, 1024]");
    if (c->num_blocks < 1 || c->num_blocks > ((int64_t(1) << 31) - 1) / c->block_size)
        return bad("num_blocks must be positive and num_blocks * block_size below 2^31");
    if (!c->k || !c->v || !c->k_scale || !c->v_scale) return bad("null cache pointer");
    if ((reinterpret_cast<uintptr_t>(c->k) | reinterpret_cast<uintptr_t>(c->v)) % 16 ||
        (reinterpret_cast<uintptr_t>(c->k_scale) | reinterpret_cast<uintptr_t>(c->v_scale)) % 4)
        return bad("misaligned cache pointer");
    out->k = static_cast<uint8_t*>(c->k);
    out->v = static_cast<uint8_t*>(c->v);
    out->k_scale = c->k_scale;
    out->v_scale = c->v_scale;
    out->num_blocks = static_cast<int>(c->num_blocks);
    out->kv_heads = static_cast<int>(c->kv_heads);
    out->block_log2 = __builtin_ctzll(static_cast<unsigned long long>(c->block_size));
    return GDSLLM_OK;
}

namespace {

// ------------------------------------------------------------------ kv_assign

constexpr int kMaxRequests = 8192;  // three words of LDS each

struct AssignArgs {
    const int32_t* lens;
    const int32_t* delta;
    int32_t* tables;
    int32_t* ring;
    const int32_t* state;
    int32_t *slots, *positions, *starts, *lens_out, *state_out;
    int64_t ld_table;
    int n, width, ring_size, block_log2, max_tokens;
};

// Every workgroup takes the sums over all requests for itself (at most 8192 of
// them: cheaper than a second launch or a grid barrier) and then writes its share
// of the tables and of the token rows.  All of it is latency (a launch takes 1.65 us):
// lengths, one scan of tokens, new and returned blocks, a ring entry, a store.  64
// decoding requests 4.9 us in a graph (called one by one, the host takes 7),
// 2048 mixed ones with 66000 token rows 7.6 us.
template <int THREADS>
__global__ __launch_bounds__(THREADS) void kv_assign(AssignArgs a) {
    extern __shared__ int32_t lds[];
    int32_t* ends = lds;              // tokens up to and with request r, at most max_tokens + 1
    int32_t* first = lds + a.n;       // blocks taken before request r; -1 where it is not served
    int32_t* given = lds + 2 * a.n;   // blocks given back before request r
    constexpr int WAVES = THREADS / 64;
    __shared__ uint64_t part[3][WAVES];
    __shared__ int taken, returned;
    const int bs = 1 << a.block_log2, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int64_t row_tokens = static_cast<int64_t>(a.width) << a.block_log2;
    auto len_of = [&](int r) { return max(a.lens[r], 0); };
    auto add_of = [&](int r) { return max(a.delta[r], 0); };
    auto drop_of = [&](int r) {
        return static_cast<int>(min(static_cast<int64_t>(len_of(r)), max(-static_cast<int64_t>(a.delta[r]), int64_t(0))));
    };
    // entry `i` (at most ring_size) behind `head`
    auto ring_at = [&](int head, int i) {
        const int64_t at = static_cast<int64_t>(head) + i;
        return at < a.ring_size ? at : at < 2 * static_cast<int64_t>(a.ring_size) ? at - a.ring_size : 0;
    };
    auto blocks = [&](int64_t t) { return static_cast<int>((t + bs - 1) >> a.block_log2); };
    // New blocks of request r, -1 where its row is too short.  Its tokens may still
    // lie behind max_tokens; then so do all later ones', and none of them is served.
    auto need_of = [&](int r) {
        const int add = add_of(r);
        const int64_t after = static_cast<int64_t>(len_of(r)) + add;
        return add == 0 ? 0 : after <= row_tokens ? blocks(after) - blocks(len_of(r)) : -1;
    };

    const int per = (a.n + THREADS - 1) / THREADS, r0 = min(tid * per, a.n), r1 = min(r0 + per, a.n);
    const int head0 = a.state[0], count0 = a.state[1];
    if (tid == 0) taken = 0;
    uint64_t tokens = 0, need = 0, back = 0;
    for (int r = r0; r < r1; ++r) {
        tokens += add_of(r);
        need += max(need_of(r), 0);
        back += blocks(len_of(r)) - blocks(len_of(r) - drop_of(r));
    }
    uint64_t at = wave_scan(tokens), upto = wave_scan(need), back_at = wave_scan(back);
    if (lane == 63) {
        part[0][wave] = at;
        part[1][wave] = upto;
        part[2][wave] = back_at;
    }
    __syncthreads();
    for (int w = 0; w < wave; ++w) {
        at += part[0][w];
        upto += part[1][w];
        back_at += part[2][w];
    }
    if (tid == THREADS - 1) returned = static_cast<int>(min(back_at, static_cast<uint64_t>(a.ring_size)));
    at -= tokens;
    upto -= need;
    back_at -= back;
    const int head = min(max(head0, 0), a.ring_size - 1), count = min(max(count0, 0), a.ring_size);
    int most = 0;
    for (int r = r0; r < r1; ++r) {
        at += add_of(r);
        const int n = need_of(r);
        const bool served = n == 0 ? add_of(r) == 0 || at <= static_cast<uint64_t>(a.max_tokens)
                                   : n > 0 && at <= static_cast<uint64_t>(a.max_tokens) && upto + n <= static_cast<uint64_t>(count);
        ends[r] = static_cast<int32_t>(min(at, static_cast<uint64_t>(a.max_tokens) + 1));
        first[r] = served ? static_cast<int32_t>(min(upto, static_cast<uint64_t>(a.ring_size))) : -1;
        given[r] = static_cast<int32_t>(min(back_at, static_cast<uint64_t>(a.ring_size)));
        upto += max(n, 0);
        if (served && n > 0) most = static_cast<int>(upto);
        back_at += blocks(len_of(r)) - blocks(len_of(r) - drop_of(r));
        if (blockIdx.x == 0) {
            a.starts[r + 1] = min(ends[r], a.max_tokens);
            a.lens_out[r] = len_of(r) + (served ? add_of(r) - drop_of(r) : 0);
        }
    }
    if (most > 0) atomicMax(&taken, most);
    __syncthreads();
    const int room = a.ring_size - count;  // ring entries that a returned block may take
    if (blockIdx.x == 0 && tid == 0) {
        a.starts[0] = 0;
        a.state_out[0] = (head + taken) % a.ring_size;
        a.state_out[1] = count - taken + min(returned, room);
    }

    // New and returned blocks: the requests spread over the waves, one to a lane,
    // which copies its blocks itself where they are few (a decoding step), else the
    // whole wave does (a prompt's, an ended request's).  A request to a wave took 6.7
    // us instead of 4.9 for 64 of them, 64 of 2048 to a wave 10.7 instead of 7.6.
    constexpr int kOwn = 4;
    const int waves = static_cast<int>(gridDim.x) * WAVES, share = min((a.n + waves - 1) / waves, 64);
    for (int base = (static_cast<int>(blockIdx.x) * WAVES + wave) * share; base < a.n; base += waves * share) {
        const int r = lane < share ? base + lane : a.n;
        int n = 0, from = 0, ring = 0;  // blocks, the first one's place in the row and in the ring
        bool take = false;
        if (r < a.n) {
            const int len = len_of(r), add = add_of(r), have = blocks(len);
            take = add > 0;
            if (take) {
                n = first[r] >= 0 ? blocks(static_cast<int64_t>(len) + add) - have : 0;
                from = have;
                ring = first[r];
            } else {
                from = blocks(len - drop_of(r));
                n = max(min(min(have, a.width) - from, room - given[r]), 0);
                ring = count + given[r];
            }
        }
        auto copy = [&](int request, int block, int place, bool taken_here) {
            int32_t* entry = a.tables + request * a.ld_table + block;
            if (taken_here) *entry = a.ring[ring_at(head, place)];
            else a.ring[ring_at(head, place)] = *entry;
        };
        if (n <= kOwn)
            for (int j = 0; j < n; ++j) copy(r, from + j, ring + j, take);
        for (uint64_t many = __ballot(n > kOwn); many; many &= many - 1) {
            const int l = __builtin_ctzll(many);
            const int count_l = __builtin_amdgcn_readlane(n, l), from_l = __builtin_amdgcn_readlane(from, l);
            const int ring_l = __builtin_amdgcn_readlane(ring, l);
            const bool take_l = __builtin_amdgcn_readlane(take ? 1 : 0, l);
            for (int j = lane; j < count_l; j += 64) copy(base + l, from_l + j, ring_l + j, take_l);
        }
    }
    // token rows: the request of a row is the first whose end lies past it
    const int total = a.n > 0 ? min(ends[a.n - 1], a.max_tokens) : 0;
    for (int t = static_cast<int>(blockIdx.x) * THREADS + tid; t < a.max_tokens; t += static_cast<int>(gridDim.x) * THREADS) {
        int slot = -1, pos = -1;
        if (t < total) {
            int lo = 0, hi = a.n - 1;
            while (lo < hi) {
                const int mid = (lo + hi) >> 1;
                if (ends[mid] > t) hi = mid;
                else lo = mid + 1;
            }
            if (first[lo] >= 0) {
                const int len = len_of(lo), have = blocks(len);
                pos = len + t - (lo > 0 ? ends[lo - 1] : 0);
                const int b = pos >> a.block_log2;
                const int id = b < have ? a.tables[lo * a.ld_table + b]
                                        : a.ring[ring_at(head, first[lo] + b - have)];
                slot = (id << a.block_log2) + (pos & (bs - 1));
            }
        }
        a.slots[t] = slot;
        a.positions[t] = pos;
    }
}

// ------------------------------------------------------------------ kv_append

struct AppendArgs {
    KvCache c;
    const uint16_t *k, *v, *q;
    uint16_t* q_out;
    const int32_t *slots, *positions;
    const float *cos, *sin;
    int64_t ldk, ldv, ldq;
    int tokens, q_heads, half;  // half: channels in one half of a rotated pair; 0: no rotation
    int max_pos;
    int rows_per_group;         // token rows of a workgroup
    int groups;                 // ceil(tokens / rows_per_group)
};

// The slot of a row that is written, -1 for padding: a slot outside the
// cache, or a position that the rotation's table does not have.
__device__ __forceinline__ int slot_of(const AppendArgs& a, int t) {
    const int s = a.slots[t];
    if (s < 0 || (s >> a.c.block_log2) >= a.c.num_blocks) return -1;
    if (a.half > 0 && static_cast<uint32_t>(a.positions[t]) >= static_cast<uint32_t>(a.max_pos)) return -1;
    return s;
}

// Cosines and sines of eight channels, and their product with eight pairs: in 64
// bits, where the products are exact; then to fp32 and from there to fp16, as
// torch's own cast from 64 bits goes (a value within 2^-25 of itself of the middle
// between two fp16 values may go to the farther one).
struct Turn {
    float4_t c[2], s[2];
    __device__ __forceinline__ void load(const float* cos, const float* sin) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            c[i] = *reinterpret_cast<const float4_t*>(cos + 4 * i);
            s[i] = *reinterpret_cast<const float4_t*>(sin + 4 * i);
        }
    }
    // own c - other s of the first half's channels, own c + other s of the second's
    __device__ __forceinline__ uint4 apply(const uint4& own, const uint4& other, bool first) const {
        const uint32_t xs[4] = {own.x, own.y, own.z, own.w}, ys[4] = {other.x, other.y, other.z, other.w};
        uint32_t r[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            uint16_t h[2];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const double a = h2f((xs[i] >> (16 * j)) & 0xFFFFu), b = h2f((ys[i] >> (16 * j)) & 0xFFFFu);
                const double bs = b * static_cast<double>(s[i / 2][2 * (i & 1) + j]);
                h[j] = f2h_bits(fp32_rounded(static_cast<float>(fma(a, static_cast<double>(c[i / 2][2 * (i & 1) + j]), first ? -bs : bs))));
            }
            r[i] = h[0] | (static_cast<uint32_t>(h[1]) << 16);
        }
        return make_uint4(r[0], r[1], r[2], r[3]);
    }
};

__device__ __forceinline__ uint4 load16(const uint16_t* p) { return *reinterpret_cast<const uint4*>(p); }

// Eight channels (chunk `ch`) of a row of keys, after the rotation.
__device__ __forceinline__ uint4 load_rotated(const AppendArgs& a, const uint16_t* row, int t, int ch) {
    const uint4 own = load16(row + 8 * ch);
    const int hc = a.half >> 3;
    if (ch >= 2 * hc) return own;
    const bool lo = ch < hc;
    const uint4 other = load16(row + 8 * (lo ? ch + hc : ch - hc));
    const int64_t at = static_cast<int64_t>(a.positions[t]) * a.half + 8 * (lo ? ch : ch - hc);
    Turn turn;
    turn.load(a.cos + at, a.sin + at);
    return turn.apply(own, other, lo);
}

// New rows t0 .. t0 + n - 1 of one page and head; `low`: the lowest offset that
// they write; `rising`: their offsets rise row by row (else a slot may occur twice).
struct Run {
    const AppendArgs* a;
    const uint16_t* src;
    uint8_t* codes;
    float* scales;
    int64_t ld;
    int t0, n, page, low, head;
    bool is_k, rising;
};

// A run by `WAVES` waves (tid: this thread's number
// among theirs): the largest finite magnitude, the scale, the old codes where it
// grew, the new codes.  The rotated rows stay in registers between the two
// passes, up to kKeep chunks of eight channels to a thread.
template <bool E4M3, int D, int WAVES>
__device__ void append_run(const Run& r, int tid, float* red) {
    constexpr int C = D / 8, N = 64 * WAVES, kKeep = 4;
    const AppendArgs& a = *r.a;
    const int bl = a.c.block_log2;
    const float top = E4M3 ? kE4m3Max : kInt8Max;
    const int chunks = r.n * C;
    auto load = [&](int i) {
        const int t = r.t0 + i / C;
        const uint16_t* row = r.src + t * r.ld;
        return r.is_k && a.half > 0 ? load_rotated(a, row, t, i % C) : load16(row + 8 * (i % C));
    };
    float amax = 0.f;
    auto largest = [&](const uint4& x) {
        const uint32_t ws[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const uint32_t h = (ws[j / 2] >> (16 * (j & 1))) & 0x7FFFu;
            amax = fmaxf(amax, h < 0x7C00u ? h2f(h) : 0.f);
        }
    };
    uint4 keep[kKeep];
#pragma unroll
    for (int j = 0; j < kKeep; ++j)
        if (tid + N * j < chunks) {
            keep[j] = load(tid + N * j);
            largest(keep[j]);
        }
    for (int i = tid + N * kKeep; i < chunks; i += N) largest(load(i));
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor(amax, o));
    if constexpr (WAVES > 1) {
        __syncthreads();
        if ((tid & 63) == 0) red[tid >> 6] = amax;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < WAVES; ++w) amax = fmaxf(amax, red[w]);
    }
    // smallest power of two with amax <= top * scale
    float want = 0x1p-32f;
    if (amax > 0.f) {
        int e;
        const float m = frexpf(amax / top, &e);
        want = fmaxf(want, ldexpf(1.f, m == 0.5f ? e - 1 : e));
    }
    const int64_t sc = static_cast<int64_t>(r.page) * a.c.kv_heads + r.head;
    const float was = r.low > 0 ? r.scales[sc] : 0.f;
    const float now = fmaxf(was, want);
    if constexpr (WAVES > 1) __syncthreads();  // every wave has read the old scale
    uint8_t* base = r.codes + ((sc << bl) * D);
    if (tid == 0) r.scales[sc] = now;
    if (r.low > 0 && was != now) {
        const float ratio = was / now;
        for (int i = tid; i < r.low * C; i += N) {
            uint2* p = reinterpret_cast<uint2*>(base + 8 * static_cast<int64_t>(i));
            const uint2 w = *p;
            float x[4], y[4];
            codes_to_f32<E4M3>(w.x, x);
            codes_to_f32<E4M3>(w.y, y);
            *p = make_uint2(to_codes<E4M3>(x[0] * ratio, x[1] * ratio, x[2] * ratio, x[3] * ratio),
                            to_codes<E4M3>(y[0] * ratio, y[1] * ratio, y[2] * ratio, y[3] * ratio));
        }
    }
    const float inv = 1.f / now;
    auto store = [&](int i, const uint4& x) {
        const int t = r.t0 + i / C, s = a.slots[t];
        if (!r.rising) {  // the last row of a slot that occurs twice is the one that stays
            for (int u = t + 1; u < r.t0 + r.n; ++u)
                if (a.slots[u] == s) return;
        }
        const uint32_t ws[4] = {x.x, x.y, x.z, x.w};
        float y[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) y[j] = h2f((ws[j / 2] >> (16 * (j & 1))) & 0xFFFFu) * inv;
        *reinterpret_cast<uint2*>(base + (s & ((1 << bl) - 1)) * D + 8 * (i % C)) =
            make_uint2(to_codes<E4M3>(y[0], y[1], y[2], y[3]), to_codes<E4M3>(y[4], y[5], y[6], y[7]));
    };
#pragma unroll
    for (int j = 0; j < kKeep; ++j)
        if (tid + N * j < chunks) store(tid + N * j, keep[j]);
    for (int i = tid + N * kKeep; i < chunks; i += N) store(i, load(i));
}

// Workgroups [0, groups * kv_heads * 2): keys (even) or values (odd) of one
// head in `rows_per_group` (at most 62) token rows.  A page's tokens stand in
// consecutive rows; the workgroup takes every page whose first row lies in its
// rows, to that page's last row wherever it is, so one workgroup alone writes a
// page.  Pages with few new rows go to one wave each, others to all of them.
// Bound by the bytes of k, v, q and the codes for prompts (2 x 1000 tokens of 32 heads
// 66 MB in 21 us, 3.1 TB/s; 8192 tokens with 32 query heads of 256 296 MB in 88 us,
// 3.4), by latency for a decode step (32 tokens 4.2 us: slot, row and scale, a maximum,
// a store).
template <bool E4M3, int D, int WAVES>
__device__ void append_pages(const AppendArgs& a, int unit) {
    __shared__ float red[WAVES];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), bl = a.c.block_log2;
    Run r;
    r.a = &a;
    r.is_k = (unit & 1) == 0;
    r.head = (unit >> 1) % a.c.kv_heads;
    r.src = (r.is_k ? a.k : a.v) + r.head * D;
    r.ld = r.is_k ? a.ldk : a.ldv;
    r.codes = r.is_k ? a.c.k : a.c.v;
    r.scales = r.is_k ? a.c.k_scale : a.c.v_scale;
    const int base = (unit >> 1) / a.c.kv_heads * a.rows_per_group - 1;  // lane 0's row: the one before the group
    const int t = base + lane, mask = (1 << bl) - 1;
    const int s = t >= 0 && t < a.tokens ? slot_of(a, t) : -1, before = __shfl_up(s, 1);
    const bool goes_on = lane > 0 && s >= 0 && before >= 0 && (s >> bl) == (before >> bl);
    const uint64_t same = __ballot(goes_on), falls = __ballot(goes_on && s <= before);
    uint64_t heads = __ballot(lane > 0 && lane <= a.rows_per_group && s >= 0 && !goes_on);
    for (int k = 0; heads; ++k, heads &= heads - 1) {
        const int l = __builtin_ctzll(heads);
        const uint64_t rest = l < 63 ? ~(same >> (l + 1)) : 1ull;
        const int more = min(__builtin_ctzll(rest), 63 - l);
        const uint64_t run = (more == 63 ? ~0ull : ((1ull << (more + 1)) - 1)) << l;
        r.t0 = base + l;
        r.n = more + 1;
        r.page = __builtin_amdgcn_readlane(s, l) >> bl;
        int low = run >> lane & 1 ? s & mask : mask;
        r.rising = !(falls & run);
        if (l + more == 63) {  // past the rows that the wave holds
            for (;;) {
                const int u = r.t0 + r.n + lane, v = u < a.tokens ? slot_of(a, u) : -1, w = u <= a.tokens ? slot_of(a, u - 1) : -1;
                const uint64_t out = ~__ballot(v >= 0 && (v >> bl) == r.page);
                const int got = out ? __builtin_ctzll(out) : 64;
                if (lane < got) low = min(low, v & mask);
                if (__ballot(lane < got && v <= w)) r.rising = false;
                r.n += got;
                if (got < 64) break;
            }
        }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) low = min(low, __shfl_xor(low, o));
        r.low = __builtin_amdgcn_readfirstlane(low);
        if (WAVES == 1 || r.n * (D / 8) > 4 * 64) append_run<E4M3, D, WAVES>(r, tid, red);
        else if (k % WAVES == wave) append_run<E4M3, D, 1>(r, lane, red);
    }
}

// The rotation of q, a token to a workgroup at a time; a thread keeps to one
// chunk of the heads' channels.
template <int D>
__device__ void rotate_q(const AppendArgs& a, int first, int step) {
    constexpr int C = D / 8;
    const int tid = threadIdx.x, ch = tid % C, hc = a.half >> 3, per = blockDim.x / C;
    const bool turns = ch < 2 * hc, lo = ch < hc;
    for (int t = first; t < a.tokens; t += step) {
        const bool live = slot_of(a, t) >= 0;
        Turn turn;
        if (turns && live) {
            const int64_t at = static_cast<int64_t>(a.positions[t]) * a.half + 8 * (lo ? ch : ch - hc);
            turn.load(a.cos + at, a.sin + at);
        }
        const uint16_t* row = a.q + t * a.ldq + 8 * ch;
        uint16_t* out = a.q_out + static_cast<int64_t>(t) * a.q_heads * D + 8 * ch;
#pragma unroll 2
        for (int h = tid / C; h < a.q_heads; h += per) {
            uint4 x = make_uint4(0, 0, 0, 0);
            if (live) {
                x = load16(row + h * D);
                if (turns) x = turn.apply(x, load16(row + h * D + 8 * (lo ? hc : -hc)), lo);
            }
            *reinterpret_cast<uint4*>(out + h * D) = x;
        }
    }
}

template <int D>
__global__ __launch_bounds__(256) void kv_rotate(AppendArgs a) {
    rotate_q<D>(a, blockIdx.x, gridDim.x);
}

template <bool E4M3, int D, int WAVES>
__global__ __launch_bounds__(WAVES * 64, WAVES == 4 ? 3 : 4) void kv_append(AppendArgs a) {
    // workgroups go to the eight XCDs in turn: each XCD takes a run of units, so
    // that those in which a page begins (every fourth, say) fall to all of them
    const int per = (a.groups * a.c.kv_heads * 2 + 7) / 8, b = blockIdx.x;
    if (b >= 8 * per) {
        rotate_q<D>(a, b - 8 * per, gridDim.x - 8 * per);
        return;
    }
    const int unit = b % 8 * per + b / 8;
    if (unit < a.groups * a.c.kv_heads * 2) append_pages<E4M3, D, WAVES>(a, unit);
}

}  // namespace
}  // namespace gdsllm

using namespace gdsllm;

extern "C" int gdsllm_kv_assign(const int32_t* lens, const int32_t* delta, int64_t requests, int32_t* block_tables,
                                int64_t table_width, int64_t ld_table, int32_t* free_ring, int64_t ring_size,
                                const int32_t* free_state, int64_t block_size, int64_t max_tokens, int32_t* slots,
                                int32_t* positions, int32_t* starts, int32_t* lens_out, int32_t* state_out,
                                void* stream) {
    const std::string n = "kv_assign";
    auto bad = [&](const std::string& m) { return set_error(GDSLLM_ERR_INVALID_ARGUMENT, n + ": " + m); };
    if (requests < 1 || requests > kMaxRequests) return bad("requests must be in [1, 8192]");
    if (block_size < 16 || block_size > 256 || (block_size & (block_size - 1)))
        return bad("block_size must be 16, 32, 64, 128 or 256, got " + std::to_string(block_size));
    if (table_width < 1 || ld_table < table_width) return bad("ld_table < table_width or an empty table");
    if (table_width > ((int64_t(1) << 31) - 1) / block_size) return bad("table_width too large");
    if (ring_size < 1 || ring_size > ((int64_t(1) << 31) - 1) / block_size)
        return bad("ring_size must be positive and ring_size * block_size below 2^31");
    if (max_tokens < 0 || max_tokens > (int64_t(1) << 30)) return bad("max_tokens must be in [0, 2^30]");
    if (!lens || !delta || !block_tables || !free_ring || !free_state || !starts || !lens_out || !state_out ||
        (max_tokens > 0 && (!slots || !positions)))
        return bad("null pointer");
    if ((reinterpret_cast<uintptr_t>(lens) | reinterpret_cast<uintptr_t>(delta) |
         reinterpret_cast<uintptr_t>(block_tables) | reinterpret_cast<uintptr_t>(free_ring) |
         reinterpret_cast<uintptr_t>(free_state) | reinterpret_cast<uintptr_t>(slots) |
         reinterpret_cast<uintptr_t>(positions) | reinterpret_cast<uintptr_t>(starts) |
         reinterpret_cast<uintptr_t>(lens_out) | reinterpret_cast<uintptr_t>(state_out)) % 4)
        return bad("misaligned pointer");
    for (const int32_t* in : {lens, delta, free_state})
        if (lens_out == in || state_out == in) return bad("lens_out and state_out must not be the inputs");
    if (lens_out == state_out) return bad("lens_out and state_out must not be one buffer");
    AssignArgs a{lens, delta, block_tables, free_ring, free_state, slots, positions, starts, lens_out, state_out,
                 ld_table, static_cast<int>(requests), static_cast<int>(table_width), static_cast<int>(ring_size),
                 __builtin_ctzll(static_cast<unsigned long long>(block_size)), static_cast<int>(max_tokens)};
    const size_t lds = 3 * sizeof(int32_t) * static_cast<size_t>(requests);
    const int threads = requests <= 256 ? 256 : 1024;
    const int64_t want = std::max((max_tokens + threads - 1) / threads, (requests + 255) / 256);
    const unsigned grid = static_cast<unsigned>(std::min<int64_t>(std::max<int64_t>(want, 1), cu_count()));
    if (threads == 256) {
        hipLaunchKernelGGL(kv_assign<256>, dim3(grid), dim3(256), lds, as_stream(stream), a);
    } else {
        if (int rc = prepare_lds(reinterpret_cast<const void*>(&kv_assign<1024>), lds)) return rc;
        hipLaunchKernelGGL(kv_assign<1024>, dim3(grid), dim3(1024), lds, as_stream(stream), a);
    }
    if (int rc = check_hip(hipGetLastError(), "kv_assign launch")) return rc;
    return ok();
}

extern "C" int gdsllm_kv_append(const gdsllm_kv_cache8* cache, const void* k, int64_t ldk, const void* v, int64_t ldv,
                                const int32_t* slots, int64_t tokens, const void* q, int64_t ldq, void* q_out,
                                int64_t q_heads, const int32_t* positions, const float* cos, const float* sin,
                                int64_t rotary, int64_t max_pos, void* stream) {
    const std::string n = "kv_append";
    auto bad = [&](const std::string& m) { return set_error(GDSLLM_ERR_INVALID_ARGUMENT, n + ": " + m); };
    AppendArgs a{};
    if (int rc = kv_cache_args(cache, n, &a.c)) return rc;
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
    a.q = static_cast<const uint16_t*>(q);
    a.q_out = static_cast<uint16_t*>(q_out);
    a.slots = slots;
    a.positions = positions;
    a.cos = cos;
    a.sin = sin;
    a.ldk = ldk;
    a.ldv = ldv;
    a.ldq = ldq;
    a.tokens = static_cast<int>(tokens);
    a.q_heads = static_cast<int>(q_heads);
    a.half = static_cast<int>(rotary / 2);
    a.max_pos = static_cast<int>(max_pos);
    // as many waves as hold a page of one head in registers; most of a prompt's
    // rows begin no page, a decoding batch's all do
    const int64_t chunks = cache->block_size * D / 8;
    const int waves = chunks <= 256 ? 1 : chunks <= 1024 ? 4 : 16;
    const int64_t share = tokens * cache->kv_heads * 2 / 512;  // rows that leave two workgroups to a compute unit
    a.rows_per_group = static_cast<int>(std::min<int64_t>(std::max<int64_t>(share, 1), std::min<int64_t>(cache->block_size, 62)));
    a.groups = static_cast<int>((tokens + a.rows_per_group - 1) / a.rows_per_group);
    const int64_t units = (static_cast<int64_t>(a.groups) * cache->kv_heads * 2 + 7) / 8 * 8;
    // q rides along, but not that of long prompts in workgroups of 1024 threads, which
    // turn a token at a time (32 heads of 256: 400 tokens 14 us riding along, 18 in a
    // launch of its own; 1600 tokens 24 and 27; 3200 tokens 41 and 35)
    const int64_t q_tokens = q ? std::min<int64_t>(tokens, 16 * static_cast<int64_t>(cu_count())) : 0;
    const bool apart = q_tokens > 2048 && waves == 16;
    const int64_t q_groups = apart ? 0 : q_tokens;
    if ((units + q_groups) * 64 * waves >= (int64_t(1) << 32)) return bad("too many tokens and heads for one call");
    const dim3 grid(static_cast<unsigned>(units + q_groups));
    const bool e4m3 = cache->format == GDSLLM_KV_E4M3;
    const hipStream_t s = as_stream(stream);
#define GDSLLM_APPEND(DIM, W)                                                                    \
    if (D == DIM && waves == W) {                                                                \
        if (e4m3) hipLaunchKernelGGL((kv_append<true, DIM, W>), grid, dim3(64 * W), 0, s, a);    \
        else hipLaunchKernelGGL((kv_append<false, DIM, W>), grid, dim3(64 * W), 0, s, a);        \
        if (apart) hipLaunchKernelGGL(kv_rotate<DIM>, dim3(static_cast<unsigned>(q_tokens)), dim3(256), 0, s, a); \
    }
    GDSLLM_APPEND(64, 1)
    GDSLLM_APPEND(64, 4)
    GDSLLM_APPEND(64, 16)
    GDSLLM_APPEND(128, 1)
    GDSLLM_APPEND(128, 4)
    GDSLLM_APPEND(128, 16)
    GDSLLM_APPEND(256, 4)
    GDSLLM_APPEND(256, 16)
#undef GDSLLM_APPEND
    if (int rc = check_hip(hipGetLastError(), "kv_append launch")) return rc;
    return ok();
}
