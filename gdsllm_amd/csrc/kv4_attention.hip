// Attention over the 4-bit KV cache (kv4_cache.hip writes it).
//
// For query row t of request b (n_b rows in this call, len_b tokens held) and
// query head h of kv head h / G:
//   x_j = scale * (q . k_j),  j <= len_b - n_b + t,   o = sum_j e^x_j v_j / sum_j e^x_j
// in one pass over the tokens with a running reference m: with y_j = x_j log2 e and
// m 7 to 11 below the largest y_j so far, acc += 2^(y_j - m) v_j, l += 2^(y_j - m).
// Elements k, v = fp16(code * scale + bias) enter the matrix cores as the fp16
// values that they are by definition: nothing of the format is left for the sums.
// Weights are rounded to fp16 for the product with v and for it alone: half an
// fp16 step of a weight, and 2^-25 at least where the largest is 2^7 to 2^11.
//
// A code becomes an element in three packed instructions for two of them: below
// the exponent of 1024 (64 for the high one of two neighbours) it is a number, less
// that exponent it is exact, and one fused multiply-add makes and rounds the
// element.

#include "kv4_cache.h"
#include "kv_attend.h"

namespace gdsllm {
namespace {

typedef AttendArgs<Kv4Cache> Args4;

__device__ __forceinline__ uint32_t bits(half2_t x) { return __builtin_bit_cast(uint32_t, x); }

// Scales and biases of two tokens side by side.
__device__ __forceinline__ half2_t scales2(uint32_t a0, uint32_t a1) {
    return __builtin_bit_cast(half2_t, __builtin_amdgcn_perm(a1, a0, 0x05040100u));
}
__device__ __forceinline__ half2_t biases2(uint32_t a0, uint32_t a1) {
    return __builtin_bit_cast(half2_t, __builtin_amdgcn_perm(a1, a0, 0x07060302u));
}
// Channels 0 .. 7 of two tokens' dwords of codes, as token pairs: f[channel].
__device__ __forceinline__ void token_pairs(const NibUnpack& n, uint32_t t0, uint32_t t1, half2_t s, half2_t b, uint32_t (&f)[8]) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const uint32_t w = __builtin_amdgcn_perm(t1, t0, h ? 0x07060302u : 0x05040100u), w8 = w >> 8;
        f[4 * h] = bits(element2(codes_low(n, w), s, b));
        f[4 * h + 1] = bits(element2(codes_high(n, w), s, b));
        f[4 * h + 2] = bits(element2(codes_low(n, w8), s, b));
        f[4 * h + 3] = bits(element2(codes_high(n, w8), s, b));
    }
}

// 16 rows over blocks [block0, block1) of a sequence, by NW waves.  Matrix tiles
// are 16x16x32 and nothing passes through LDS but the block table and the waves'
// sums:
//  * scores S^T = K Q^T: lane l gives key row l % 16 and a quarter of its channels
//    (one 16-byte load for each 128, all in one group: one scale and bias), eight
//    of them, in the order their conversion gives, to a step; Q's operand takes the
//    same order.  It receives, for query l % 16, tokens 4 * group .. + 3 of each 16;
//  * O^T = V^T P^T: its B operand is exactly those eight weights of two score
//    tiles, in place; V's operand needs eight tokens of one channel in a lane: lanes
//    load D/16 channels of the eight tokens and pair two tokens' halves of a dword
//    with v_perm before the conversion.
template <int D, int NW_>
struct RowTile4 {
    typedef Args4 Args;
    static constexpr int kRows = 16, kD = D, kPerCu = per_cu(D);
    static constexpr int kThreads = NW_ * 64;
    static constexpr int NT = 2;        // score tiles of an iteration
    static constexpr int NW = NW_;
    static constexpr int KS = D / 32;   // score steps of 32 channels, a dword of codes to a lane each
    static constexpr int KW = D == 256 ? 2 : 1;  // 16-byte (D = 64: 8-byte) loads of keys, a group each
    static constexpr int DB = D / 16;   // channels of V a lane holds
    static constexpr int VW = (DB + 7) / 8;  // dwords of them
    static constexpr int TT = 16 * NT;  // tokens of an iteration
    struct Codes {
        uint32_t k[NT][KS], ka[NT][KW];
        uint32_t v[NT][4][VW];
        u32x4_t va[NT];
    };
    struct Lds {
        int id[kMaxPages];
        int none[kMaxPages];
        float m[NW][16], l[NW][16];
        float o[NW][16][D + 4];
    };
    // First channel of a lane's dword i.
    __device__ __forceinline__ static int channel(int i, int g) { return D == 64 ? 16 * g + 8 * i : 128 * (i / 4) + 32 * g + 8 * (i % 4); }

    __device__ static void run(const Args& a, Lds& s, int b, const Rows<16>& R, int tile, int head, int block0, int block1,
                               int slot, int early) {
        const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), col = lane & 15,
                  g = lane >> 4;
        const int bl = a.c.block_log2;
        const NibUnpack nib;
        // byte offsets of a lane's codes from its token row's, and of its affine pairs' groups
        const uint32_t klane = col * (D / 2) + channel(0, g) / 2, vlane = 4 * g * (D / 2) + col * DB / 2;
        int kgroup[KW];
#pragma unroll
        for (int i = 0; i < KW; ++i) kgroup[i] = channel(4 * i, g) >> a.c.group_log2;
        const int vgroup = col * DB >> a.c.group_log2;
        const int k0 = block0 * kBlock, k1 = min(block1 * kBlock, R.keys(a, tile * 16, 16));
        const int r = tile * 16 + col;
        const bool valid = r < R.rows;
        const int t_row = R.start + (valid ? r / a.group : 0), h_row = head * a.group + (valid ? r % a.group : 0);
        const int last = valid ? R.len - R.n + r / a.group : -1;  // last key this row sees
        const int all_see = R.len - R.n + tile * 16 / a.group;    // every row sees keys up to here

        half8_t qf[KS];
#pragma unroll
        for (int i = 0; i < KS; ++i) {
            uint4 w = make_uint4(0, 0, 0, 0);
            if (valid) w = *reinterpret_cast<const uint4*>(a.q + t_row * a.ldq + h_row * D + channel(i, g));
            qf[i] = __builtin_bit_cast(half8_t, pairs_from_rising(w));
        }
        float4_t acc[DB];
#pragma unroll
        for (int j = 0; j < DB; ++j) acc[j] = float4_t{0.f, 0.f, 0.f, 0.f};
        float m = -INFINITY, l = 0.f;

        if (k1 <= k0) lds_barrier();
        for (int seg = k0; seg < k1; seg += kSegment) {
            const int seg_end = min(seg + kSegment, k1);
            const int p0 = seg >> bl, pages = ((min(seg + kSegment, (k1 + TT - 1) & ~(TT - 1)) - 1) >> bl) - p0 + 1;
            lds_barrier();  // the last segment's table, or the last sequence's sums, have been read
            bool lost = false;
            for (int p = tid; p < pages; p += NW * 64) {
                const int page = p0 + p;
                int id = -1;
                if (page < a.width && (page << bl) < k1) id = early != -2 && seg == 0 ? early : a.tables[b * a.ld_table + page];
                const bool ok = id >= 0 && id < a.c.num_blocks;
                s.id[p] = ok ? id : 0;
                s.none[p] = !ok;
                lost |= !ok && (page << bl) < k1;
            }
            const bool some_lost = __syncthreads_or(lost);
            // A tile's first token among the pool's (block, head) runs, and within its block.
            auto run_of = [&](int token) {
                return static_cast<int64_t>(__builtin_amdgcn_readfirstlane(s.id[(token >> bl) - p0])) * a.c.kv_heads + head;
            };
            auto off_of = [&](int token) { return token & ((1 << bl) - 1); };
            auto load_k = [&](Codes& w, int t, int token) {
                const int64_t run = run_of(token);
                const uint8_t* p = a.c.k + ((run << bl) + off_of(token)) * (D / 2) + klane;
                const uint32_t* pa = a.c.k_affine + ((run * a.c.groups) << bl) + off_of(token) + col;
#pragma unroll
                for (int i = 0; i < KW; ++i) {
                    if constexpr (D == 64) {
                        const uint64_t x = __builtin_nontemporal_load(reinterpret_cast<const uint64_t*>(p));
                        w.k[t][0] = static_cast<uint32_t>(x);
                        w.k[t][1] = static_cast<uint32_t>(x >> 32);
                    } else {
                        const u32x4_t x = __builtin_nontemporal_load(reinterpret_cast<const u32x4_t*>(p + 64 * i));
#pragma unroll
                        for (int j = 0; j < 4; ++j) w.k[t][4 * i + j] = x[j];
                    }
                    w.ka[t][i] = __builtin_nontemporal_load(pa + (kgroup[i] << bl));
                }
            };
            auto load_v = [&](Codes& w, int t, int token) {
                const int64_t run = run_of(token);
                const uint8_t* p = a.c.v + ((run << bl) + off_of(token)) * (D / 2) + vlane;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint8_t* pi = p + i * (D / 2);
                    if constexpr (D == 64) {
                        w.v[t][i][0] = __builtin_nontemporal_load(reinterpret_cast<const uint16_t*>(pi));
                    } else if constexpr (D == 128) {
                        w.v[t][i][0] = __builtin_nontemporal_load(reinterpret_cast<const uint32_t*>(pi));
                    } else {
                        const uint64_t x = __builtin_nontemporal_load(reinterpret_cast<const uint64_t*>(pi));
                        w.v[t][i][0] = static_cast<uint32_t>(x);
                        w.v[t][i][VW - 1] = static_cast<uint32_t>(x >> 32);
                    }
                }
                w.va[t] = __builtin_nontemporal_load(reinterpret_cast<const u32x4_t*>(
                    a.c.v_affine + ((run * a.c.groups + vgroup) << bl) + off_of(token) + 4 * g));
            };
            constexpr int step = NW * TT;
            int base = seg + wave * TT;
            Codes w;
            if (base < seg_end) {
#pragma unroll
                for (int t = 0; t < NT; ++t) load_k(w, t, base + 16 * t);
#pragma unroll
                for (int t = 0; t < NT; ++t) load_v(w, t, base + 16 * t);
            }
            for (; base < seg_end; base += step) {
                const bool more = base + step < seg_end;
                float x[NT][4];
                float mx = -INFINITY;
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    float4_t sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int i = 0; i < KS; ++i) {
                        const half8_t kf = __builtin_bit_cast(half8_t, elements8(nib, w.k[t][i], w.ka[t][i / 4]));
                        sum = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, qf[i], sum, 0, 0, 0);
                    }
#pragma unroll
                    for (int i = 0; i < 4; ++i) x[t][i] = sum[i] * a.scale_log2;
                }
                if (more) {  // the keys' registers are free: the next tile's
#pragma unroll
                    for (int t = 0; t < NT; ++t) load_k(w, t, base + step + 16 * t);
                }
                if (base + TT - 1 > all_see || base + TT > k1 || some_lost) {
#pragma unroll
                    for (int t = 0; t < NT; ++t) {
                        // a block outside the cache has no weight
                        const bool none = s.none[((base + 16 * t) >> bl) - p0];
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const int j = base + 16 * t + 4 * g + i;
                            if (j > last || j >= k1 || none) x[t][i] = -INFINITY;
                            if (j >= k1 || none) w.va[t][i] = 0;  // what lies there may be no number
                        }
                    }
                }
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int i = 0; i < 4; ++i) mx = fmaxf(mx, x[t][i]);
                mx = over_groups(mx, [](float u, float v) { return fmaxf(u, v); });
                // the reference follows the maximum only when a weight would pass 2^kMost
                if (__any(mx - m > kMost)) {
                    const float m_new = fmaxf(m, mx - kSet);
                    const float alpha = __builtin_amdgcn_exp2f(m - (m_new == -INFINITY ? 0.f : m_new));
                    l *= alpha;
#pragma unroll
                    for (int j = 0; j < DB; ++j) acc[j] *= alpha;
                    m = m_new;
                }
                const float ref = m == -INFINITY ? 0.f : m;
                half8_t pf[NT / 2];
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float p = __builtin_amdgcn_exp2f(x[t][i] - ref);
                        l += p;
                        pf[t / 2][4 * (t & 1) + i] = static_cast<half_t>(p);
                    }
#pragma unroll
                for (int u = 0; u < NT / 2; ++u)
#pragma unroll
                    for (int c = 0; c < VW; ++c) {
                        uint32_t f[4][8];  // [token pair][channel]
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            const int t = 2 * u + k / 2, i = 2 * (k & 1);
                            token_pairs(nib, w.v[t][i][c], w.v[t][i + 1][c], scales2(w.va[t][i], w.va[t][i + 1]),
                                        biases2(w.va[t][i], w.va[t][i + 1]), f[k]);
                        }
#pragma unroll
                        for (int j = 0; j < (DB < 8 ? DB : 8); ++j) {
                            const half8_t vf = __builtin_bit_cast(half8_t, make_uint4(f[0][j], f[1][j], f[2][j], f[3][j]));
                            acc[8 * c + j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, pf[u], acc[8 * c + j], 0, 0, 0);
                        }
                    }
                if (more) {
#pragma unroll
                    for (int t = 0; t < NT; ++t) load_v(w, t, base + step + 16 * t);
                }
            }
        }
        l = over_groups(l, [](float u, float v) { return u + v; });

        // the waves' sums meet in LDS; every thread adds four channels of a row
        if (g == 0) {
            s.m[wave][col] = m;
            s.l[wave][col] = l;
        }
        if (valid) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < DB; j += 4)
                    *reinterpret_cast<float4_t*>(&s.o[wave][col][(4 * g + i) * DB + j]) =
                        float4_t{acc[j][i], acc[j + 1][i], acc[j + 2][i], acc[j + 3][i]};
        }
        lds_barrier();
        const int count = min(16, R.rows - tile * 16);
        for (int i = tid; i < count * (D / 4); i += NW * 64) {
            const int rr = i / (D / 4), d = 4 * (i % (D / 4));
            float mw = s.m[0][rr];
#pragma unroll
            for (int w = 1; w < NW; ++w) mw = fmaxf(mw, s.m[w][rr]);
            const float ref = mw == -INFINITY ? 0.f : mw;
            float lw = 0.f;
            float4_t o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int w = 0; w < NW; ++w) {
                const float f = __builtin_amdgcn_exp2f(s.m[w][rr] - ref);
                lw = fmaf(s.l[w][rr], f, lw);
                o += *reinterpret_cast<const float4_t*>(&s.o[w][rr][d]) * f;
            }
            if (slot < 0) {
                const float inv = inverse(lw);
                const int row = tile * 16 + rr;
                uint2 w;
                w.x = pack_h2(static_cast<half_t>(o[0] * inv), static_cast<half_t>(o[1] * inv));
                w.y = pack_h2(static_cast<half_t>(o[2] * inv), static_cast<half_t>(o[3] * inv));
                *reinterpret_cast<uint2*>(a.o + (R.start + row / a.group) * a.ldo + (head * a.group + row % a.group) * D + d) = w;
            } else {
                *reinterpret_cast<float4_t*>(a.part_o + (static_cast<int64_t>(slot) * 16 + rr) * D + d) = o;
                if (d == 0) a.part_ml[slot * 16 + rr] = make_float2(mw, lw);
            }
        }
    }
};

// 32 rows to each of NW waves over blocks [block0, block1) of a sequence, for
// prompts.  BN tokens at a time become elements once, in LDS (two buffers, one
// barrier a tile), while the tile before is worked on; matrix tiles are 32x32x16:
//  * S^T = K Q^T: K [token][channel] from LDS, each eight channels in the order
//    their conversion gives, Q in registers in that order; lane l receives, for
//    query l % 32, tokens 8b + 4h + j of each 32 (h = l / 32);
//  * O^T = V^T P^T: again those weights are the B operand in place, eight tokens
//    16u + 8(i/4) + 4h + i%4 to a lane, and V lies in LDS transposed, [channel]
//    [token], with its tokens in that order, so its operand is one 16-byte read.
// Rows of both tiles are 16 bytes longer than their data: reads and writes touch
// every bank once.
template <int D, int NW>
struct PromptTile4 {
    typedef Args4 Args;
    static constexpr int kRows = 32 * NW, kThreads = 64 * NW, kD = D, kPerCu = D == 256 ? 1 : 2;
    static constexpr int BN = D == 256 ? 32 : 64;
    static constexpr int ST = BN / 32, KS = D / 16, DT = D / 32, U = BN / 16;
    // 16-channel chunks of K, and the ones a thread converts (the last threads none where there are fewer)
    static constexpr int KR = D / 16, KT = BN * KR, KC = (KT + kThreads - 1) / kThreads;
    // (four tokens, 8 channels) pieces of V, and the ones a thread converts
    static constexpr int VQ = BN / 4, VC = VQ * (D / 8), VN = (VC + kThreads - 1) / kThreads;
    struct Lds {
        int id[kMaxPages];
        int none[kMaxPages];
        uint16_t k[2][BN][D + 8];
        uint16_t v[2][D][BN + 8];
    };
    struct Codes {
        uint64_t k[KC];
        uint32_t ka[KC];
        uint32_t v[VN][4];
        u32x4_t va[VN];
    };

    __device__ static void run(const Args& a, Lds& s, int b, const Rows<kRows>& R, int tile, int head, int block0, int block1,
                               int slot, int early) {
        const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), col = lane & 31,
                  h = lane >> 5;
        const int bl = a.c.block_log2;
        const NibUnpack nib;
        const int k0 = block0 * kBlock, k1 = min(block1 * kBlock, R.keys(a, tile * kRows, kRows));
        const int w0 = tile * kRows + wave * 32;  // this wave's rows
        const int r = w0 + col;
        const bool valid = r < R.rows;
        const int t_row = R.start + (valid ? r / a.group : 0), h_row = head * a.group + (valid ? r % a.group : 0);
        const int last = valid ? R.len - R.n + r / a.group : -1;
        const int all_see = R.len - R.n + w0 / a.group;
        const int k1w = w0 < R.rows ? min(k1, R.keys(a, w0, 32)) : 0;  // keys that this wave's rows see

        half8_t qf[KS];
#pragma unroll
        for (int i = 0; i < KS; ++i) {
            uint4 w = make_uint4(0, 0, 0, 0);
            if (valid) w = *reinterpret_cast<const uint4*>(a.q + t_row * a.ldq + h_row * D + 16 * i + 8 * h);
            qf[i] = __builtin_bit_cast(half8_t, pairs_from_rising(w));
        }
        float16_t acc[DT];
#pragma unroll
        for (int j = 0; j < DT; ++j)
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[j][i] = 0.f;
        float m = -INFINITY, l = 0.f;

        if (k1 <= k0) lds_barrier();
        for (int seg = k0; seg < k1; seg += kSegment) {
            const int seg_end = min(seg + kSegment, k1);
            const int p0 = seg >> bl, pages = ((min(seg + kSegment, (k1 + BN - 1) & ~(BN - 1)) - 1) >> bl) - p0 + 1;
            lds_barrier();
            bool lost = false;
            for (int p = tid; p < pages; p += kThreads) {
                const int page = p0 + p;
                int id = -1;
                if (page < a.width && (page << bl) < k1) id = early != -2 && seg == 0 ? early : a.tables[b * a.ld_table + page];
                const bool ok = id >= 0 && id < a.c.num_blocks;
                s.id[p] = ok ? id : 0;
                s.none[p] = !ok;
                lost |= !ok && (page << bl) < k1;
            }
            const bool some_lost = __syncthreads_or(lost);

            auto run_of = [&](int token) { return static_cast<int64_t>(s.id[(token >> bl) - p0]) * a.c.kv_heads + head; };
            auto off_of = [&](int token) { return token & ((1 << bl) - 1); };
            auto load = [&](Codes& w, int base) {
#pragma unroll
                for (int i = 0; i < KC; ++i) {
                    const int c = tid + kThreads * i, token = base + c / KR, ch = 16 * (c % KR);
                    if (KT % kThreads != 0 && c >= KT) continue;
                    const int64_t run = run_of(token);
                    w.k[i] = *reinterpret_cast<const uint64_t*>(a.c.k + ((run << bl) + off_of(token)) * (D / 2) + ch / 2);
                    w.ka[i] = a.c.k_affine[((run * a.c.groups + (ch >> a.c.group_log2)) << bl) + off_of(token)];
                }
#pragma unroll
                for (int i = 0; i < VN; ++i) {
                    const int c = tid + kThreads * i, token = base + 4 * (c % VQ), ch = 8 * (c / VQ);
                    if (VC % kThreads == 0 || c < VC) {
                        const int64_t run = run_of(token);
                        const uint8_t* p = a.c.v + ((run << bl) + off_of(token)) * (D / 2) + ch / 2;
#pragma unroll
                        for (int j = 0; j < 4; ++j) w.v[i][j] = *reinterpret_cast<const uint32_t*>(p + j * (D / 2));
                        w.va[i] = *reinterpret_cast<const u32x4_t*>(a.c.v_affine + ((run * a.c.groups + (ch >> a.c.group_log2)) << bl) + off_of(token));
                    }
                }
            };
            auto store = [&](Codes& w, int base, int buf) {
#pragma unroll
                for (int i = 0; i < KC; ++i) {
                    const int c = tid + kThreads * i;
                    if (KT % kThreads != 0 && c >= KT) continue;
                    uint4* p = reinterpret_cast<uint4*>(&s.k[buf][c / KR][16 * (c % KR)]);
                    p[0] = elements8(nib, static_cast<uint32_t>(w.k[i]), w.ka[i]);
                    p[1] = elements8(nib, static_cast<uint32_t>(w.k[i] >> 32), w.ka[i]);
                }
                const bool tail = base + BN > k1 || some_lost;
#pragma unroll
                for (int i = 0; i < VN; ++i) {
                    const int c = tid + kThreads * i, quad = c % VQ;
                    if (VC % kThreads == 0 || c < VC) {
                        if (tail) {  // what lies behind the last token, or in a lost block, may be no number
                            const int token = base + 4 * quad;
                            const bool none = s.none[(token >> bl) - p0];
#pragma unroll
                            for (int j = 0; j < 4; ++j)
                                if (none || token + j >= k1) w.va[i][j] = 0;
                        }
                        const int pos = 16 * (quad / 4) + 8 * (quad & 1) + 4 * ((quad >> 1) & 1);
                        uint32_t f[2][8];
#pragma unroll
                        for (int k = 0; k < 2; ++k)
                            token_pairs(nib, w.v[i][2 * k], w.v[i][2 * k + 1], scales2(w.va[i][2 * k], w.va[i][2 * k + 1]),
                                        biases2(w.va[i][2 * k], w.va[i][2 * k + 1]), f[k]);
#pragma unroll
                        for (int j = 0; j < 8; ++j)
                            *reinterpret_cast<uint2*>(&s.v[buf][8 * (c / VQ) + j][pos]) = make_uint2(f[0][j], f[1][j]);
                    }
                }
            };

            Codes w;
            load(w, seg);
            store(w, seg, 0);
            lds_barrier();
            int buf = 0;
            for (int base = seg; base < seg_end; base += BN, buf ^= 1) {
                const bool more = base + BN < seg_end;
                if (more) load(w, base + BN);
                if (base < k1w) {
                    float16_t x[ST];
#pragma unroll
                    for (int t = 0; t < ST; ++t) {
#pragma unroll
                        for (int i = 0; i < 16; ++i) x[t][i] = 0.f;
#pragma unroll
                        for (int i = 0; i < KS; ++i) {
                            const half8_t kf = *reinterpret_cast<const half8_t*>(&s.k[buf][32 * t + col][16 * i + 8 * h]);
                            x[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf, qf[i], x[t], 0, 0, 0);
                        }
                    }
                    if (base + BN - 1 > all_see || base + BN > k1 || some_lost) {
#pragma unroll
                        for (int t = 0; t < ST; ++t)
#pragma unroll
                            for (int i = 0; i < 16; ++i) {
                                const int j = base + 32 * t + 8 * (i / 4) + 4 * h + i % 4;
                                if (j > last || j >= k1 || (some_lost && s.none[(j >> bl) - p0])) x[t][i] = -INFINITY;
                            }
                    }
                    float mx = -INFINITY;
#pragma unroll
                    for (int t = 0; t < ST; ++t)
#pragma unroll
                        for (int i = 0; i < 16; ++i) mx = fmaxf(mx, x[t][i]);
                    {
                        float p = mx, q = mx;
                        swap32(p, q);
                        mx = fmaxf(p, q) * a.scale_log2;
                    }
                    if (__any(mx - m > kMost)) {  // as in RowTile4
                        const float m_new = fmaxf(m, mx - kSet);
                        const float alpha = __builtin_amdgcn_exp2f(m - (m_new == -INFINITY ? 0.f : m_new));
                        l *= alpha;
#pragma unroll
                        for (int j = 0; j < DT; ++j) acc[j] *= alpha;
                        m = m_new;
                    }
                    const float ref = m == -INFINITY ? 0.f : m;
#pragma unroll
                    for (int u = 0; u < U; ++u) {
                        half8_t pf;
                        float p[8];
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            p[i] = __builtin_amdgcn_exp2f(fmaf(x[u / 2][8 * (u & 1) + i], a.scale_log2, -ref));
                            pf[i] = static_cast<half_t>(p[i]);
                        }
                        l += ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
#pragma unroll
                        for (int j = 0; j < DT; ++j) {
                            const half8_t vf = *reinterpret_cast<const half8_t*>(&s.v[buf][32 * j + col][16 * u + 8 * h]);
                            acc[j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf, pf, acc[j], 0, 0, 0);
                        }
                    }
                }
                if (more) store(w, base + BN, buf ^ 1);
                lds_barrier();
            }
        }
        {
            float p = l, q = l;
            swap32(p, q);
            l = p + q;
        }
        if (!valid) return;
        if (slot < 0) {
            const float inv = inverse(l);
            uint16_t* o = a.o + t_row * a.ldo + h_row * D;
#pragma unroll
            for (int j = 0; j < DT; ++j)
#pragma unroll
                for (int i = 0; i < 16; i += 4) {
                    uint2 w;
                    w.x = pack_h2(static_cast<half_t>(acc[j][i] * inv), static_cast<half_t>(acc[j][i + 1] * inv));
                    w.y = pack_h2(static_cast<half_t>(acc[j][i + 2] * inv), static_cast<half_t>(acc[j][i + 3] * inv));
                    *reinterpret_cast<uint2*>(o + 32 * j + 2 * i + 4 * h) = w;
                }
        } else {
            const int64_t row = static_cast<int64_t>(slot) * kRows + wave * 32 + col;
#pragma unroll
            for (int j = 0; j < DT; ++j)
#pragma unroll
                for (int i = 0; i < 16; i += 4)
                    *reinterpret_cast<float4_t*>(a.part_o + row * D + 32 * j + 2 * i + 4 * h) =
                        float4_t{acc[j][i], acc[j][i + 1], acc[j][i + 2], acc[j][i + 3]};
            if (h == 0) a.part_ml[row] = make_float2(m, l);
        }
    }
};

template <int D>
int launch_attend4(Args4 a, const Plan& p, int64_t blocks, int64_t max_rows, char* workspace, hipStream_t s) {
    const char* where = "kv4_attention launch";
    const int zero_other = a.zero_other;
    a.zero_other = p.few.on ? zero_other : 0;
    if (int rc = launch_part<RowTile4<D, 8>, RowTile4<D, 4>>(a, p.few, blocks, p.many.on ? kFewRows : max_rows, workspace, s, where))
        return rc;
    a.zero_other = p.few.on ? 0 : zero_other;
    char* ws = workspace + p.few.bytes;
    if constexpr (D <= 128)
        if (p.many.rows == 256) return launch_part<PromptTile4<D, 8>, PromptTile4<D, 4>>(a, p.many, blocks, max_rows, ws, s, where);
    return launch_part<PromptTile4<D, 4>, PromptTile4<D, 4>>(a, p.many, blocks, max_rows, ws, s, where);
}

}  // namespace
}  // namespace gdsllm

using namespace gdsllm;

extern "C" size_t gdsllm_kv4_attention_workspace_size(int64_t requests, int64_t q_heads, int64_t kv_heads, int64_t head_dim,
                                                      int64_t max_new, int64_t max_len) {
    if (!attend_sizes(requests, q_heads, kv_heads, head_dim, max_new, max_len)) return 0;
    return workspace_bound(requests, q_heads, kv_heads, head_dim, max_new, max_len);
}

extern "C" int gdsllm_kv4_attention(const gdsllm_kv_cache4* cache, const void* q, int64_t ldq, void* o, int64_t ldo,
                                    int64_t tokens, int64_t q_heads, const int32_t* block_tables, int64_t table_width,
                                    int64_t ld_table, const int32_t* lens, const int32_t* starts, int64_t requests,
                                    float scale, int64_t max_new, int64_t max_len, int zero_other, void* workspace,
                                    size_t workspace_bytes, void* stream) {
    Args4 a{};
    AttendCall c;
    if (int rc = kv4_cache_args(cache, "kv4_attention", &a.c)) return rc;
    if (int rc = attend_call("kv4_attention", cache, q, ldq, o, ldo, tokens, q_heads, block_tables, table_width, ld_table, lens,
                             starts, requests, scale, max_new, max_len, zero_other, workspace, workspace_bytes, a, &c))
        return rc;
    if (c.empty) return ok();
    const hipStream_t s = as_stream(stream);
    char* ws = static_cast<char*>(workspace);
    int rc = GDSLLM_OK;
    if (cache->head_dim == 64) rc = launch_attend4<64>(a, c.plan, c.blocks, c.max_rows, ws, s);
    else if (cache->head_dim == 128) rc = launch_attend4<128>(a, c.plan, c.blocks, c.max_rows, ws, s);
    else rc = launch_attend4<256>(a, c.plan, c.blocks, c.max_rows, ws, s);
    return rc ? rc : ok();
}
