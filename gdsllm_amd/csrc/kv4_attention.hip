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
// fp16 step of a weight, and 2^-25 at least where the largest is 2^7 to 2^11.  The
// matrix instructions take fp16 on both sides; a weight as the sum of two such
// operands costs a 4096-token prompt 232 us instead of 172 and 32 decoding requests
// 47.8 instead of 44.8, for results 2.0e-4 (their own rounding) instead of 2.6e-4 from
// those in 64 bits.
//
// A code becomes an element in three packed instructions for two of them: below
// the exponent of 1024 (64 for the high one of two neighbours) it is a number, less
// that exponent it is exact, and one fused multiply-add makes and rounds the
// element.

#include <type_traits>

#include "kv4_cache.h"
#include "kv_attend.h"

namespace gdsllm {
namespace {

typedef AttendArgs<Kv4Cache> Args4;
constexpr int kPromptsPerCu = 1;  // workgroups of PromptTile4 that a compute unit holds at once

__device__ __forceinline__ uint32_t bits(half2_t x) { return __builtin_bit_cast(uint32_t, x); }

// T at `offset` bytes from a wave-uniform address: a scalar base and a 32-bit
// offset, where the compiler would keep a 64-bit address for each lane.
template <class T>
__device__ __forceinline__ T load_from(const void* base, uint32_t offset) {
    auto p = (const __attribute__((address_space(1))) char*)(base);
    asm volatile("" : "+s"(p), "+v"(offset));
    return *(const __attribute__((address_space(1))) T*)(p + offset);
}

// Scales and biases of two tokens side by side.
__device__ __forceinline__ half2_t scales2(uint32_t a0, uint32_t a1) {
    return __builtin_bit_cast(half2_t, __builtin_amdgcn_perm(a1, a0, 0x05040100u));
}
__device__ __forceinline__ half2_t biases2(uint32_t a0, uint32_t a1) {
    return __builtin_bit_cast(half2_t, __builtin_amdgcn_perm(a1, a0, 0x07060302u));
}
// Channels 4 * half .. + 3 of two tokens' dwords of codes, as token pairs: f[channel].
__device__ __forceinline__ void token_pairs(const NibUnpack& n, uint32_t t0, uint32_t t1, half2_t s, half2_t b, int half,
                                            uint32_t* f) {
    const uint32_t w = __builtin_amdgcn_perm(t1, t0, half ? 0x07060302u : 0x05040100u), w8 = w >> 8;
    f[0] = bits(element2(codes_low(n, w), s, b));
    f[1] = bits(element2(codes_high(n, w), s, b));
    f[2] = bits(element2(codes_low(n, w8), s, b));
    f[3] = bits(element2(codes_high(n, w8), s, b));
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
    // kBegin: 32 requests of up to 8192 tokens 43.6 us with 6 (49.4 with none, 44.8 with 4, 45.1 with 7), 32 of up
    // to 4000 of 256 channels 22.7 (26.9, 24.2, 24.4)
    static constexpr int kRows = 16, kD = D, kPerCu = per_cu(D), kBegin = 6;
    static constexpr bool kRowJoin = false;
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
                            const half2_t sc = scales2(w.va[t][i], w.va[t][i + 1]), bi = biases2(w.va[t][i], w.va[t][i + 1]);
                            token_pairs(nib, w.v[t][i][c], w.v[t][i + 1][c], sc, bi, 0, f[k]);
                            if constexpr (DB >= 8) token_pairs(nib, w.v[t][i][c], w.v[t][i + 1][c], sc, bi, 1, f[k] + 4);
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

// Prompts: 32 rows to each of eight waves over blocks [block0, block1) of a
// sequence, 256 rows (SPLIT 1) or 128 (SPLIT 2).  BN tokens at a time become
// elements once, in LDS; matrix tiles are 32x32x16:
//  * S^T = K Q^T: K [token][channel] from LDS, each eight channels in the order
//    their conversion gives, Q in registers (D = 256: in LDS) in that order; lane l
//    receives, for query l % 32, tokens 8b + 4h + j of each 32 (h = l / 32);
//  * O^T = V^T P^T: again those weights are the B operand in place, eight tokens
//    16u + 8(i/4) + 4h + i%4 to a lane, and V lies in LDS transposed, [channel]
//    [token], with its tokens in that order, so its operand is one 16-byte read.
// K's rows are 16 bytes longer than their data and V's chunks of eight tokens
// change places from row to row (v_place), so that reads touch every bank once
// (rows of V 16 bytes longer instead, and fewer addresses: twice the conflicts,
// 171 us for 163).
//
// Two waves share a SIMD, one of each group of four.  Time goes in slots between
// barriers: in one a group feeds the matrix cores alone (the values of its tile,
// the scores of its next one), in the next it does the vector work (softmax, the
// conversion of codes and their loads) while the other group has the matrix cores.
// With SPLIT 1 the groups have the same keys and other rows, each tile two slots, and
// each converts half of it.  With SPLIT 2 they have the same rows and
// every other tile, each tile one slot, and add their sums in the end: twice the
// conversion to a row, half the rows to a workgroup.
//
// A prompt of 4096 tokens, 32 heads of 128 channels: 163 us (four waves that
// do all of it in turn, two workgroups to a compute unit: 178), 840 TFLOP/s.  A
// slot takes 2000 cycles: its 32 matrix instructions 1024 of them, its vector work
// as many as the slot, 230 instructions for 64 tokens of 32 rows at 5 to 8 cycles.
// Beside that a workgroup takes 8 us to begin and to end, of 130, and the clock
// falls to 1.8 GHz.  Conversions among the matrix instructions of the same slot:
// 168 us, in either order of priority.
template <int D, int SPLIT>
struct PromptTile4 {
    typedef Args4 Args;
    static constexpr int kRows = 256 / SPLIT, kThreads = 512, kD = D, kPerCu = kPromptsPerCu, kBegin = 6;
    static constexpr bool kRowJoin = true;
    static constexpr int BN = D == 256 ? 32 : D == 64 && SPLIT == 1 ? 128 : 64;
    static constexpr int ST = BN / 32, KS = D / 16, DT = D / 32, U = BN / 16;
    static constexpr bool kQInLds = D == 256;
    // Threads that share the conversion of a tile: a group's, or both groups' (SPLIT 1).
    static constexpr int kConv = 512 / SPLIT;
    // 16-channel chunks of K, and the ones a thread converts
    static constexpr int KR = D / 16, KC = BN * KR / kConv;
    // pieces of V, PT tokens by eight channels: one to a thread
    static constexpr int VR = D / 8, PT = BN * VR / kConv;
    static_assert(KC >= 1 && (PT == 2 || PT == 4), "chunks fall evenly to threads");
    static_assert(64 / KR <= 16 && 64 / VR * PT <= 16, "a wave's chunks lie in one block");
    // V^T's rows in LDS are BN tokens in chunks of eight, at places that keep eight
    // neighbouring rows (reads) and every eighth row (writes) in different banks.
    __device__ __forceinline__ static int v_place(int channel, int token8) {
        if (BN == 128) return token8 ^ ((channel ^ (channel >> 4)) & 15);
        return BN == 64 ? token8 ^ ((channel ^ (channel >> 3)) & 7) : token8 ^ (((channel >> 2) ^ (channel >> 4)) & 3);
    }
    struct Tiles {
        uint16_t k[2][BN][D + 8];
        uint16_t v[2][D][BN];
        uint16_t q[kQInLds ? kRows : 1][D + 8];
    };
    struct Sums {  // of the second group, SPLIT 2
        float o[SPLIT == 2 ? kRows : 1][D + 4];
        float m[SPLIT == 2 ? kRows : 1], l[SPLIT == 2 ? kRows : 1];
    };
    struct Lds {
        int run[kMaxPages];  // a block's and head's place in the pool; -1: outside the cache
        union {
            Tiles t;
            Sums sum;
        };
    };

    __device__ static void run(const Args& a, Lds& s, int b, const Rows<kRows>& R, int tile, int head, int block0, int block1,
                               int slot, int early) {
        const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), col = lane & 31,
                  h = lane >> 5;
        const int group = wave >> 2;
        const int cw = SPLIT == 1 ? wave : wave & 3, ct = tid & (kConv - 1);  // of those that convert a tile
        const int bl = a.c.block_log2, groups_log2 = __builtin_ctz(D) - a.c.group_log2;
        const NibUnpack nib;
        const int k0 = block0 * kBlock, k1 = min(block1 * kBlock, R.keys(a, tile * kRows, kRows));
        const int wr = cw * 32;  // this wave's first row in the tile
        // a thread's chunk of K and piece of V from its wave's first token on: bytes of codes, pairs
        const uint32_t k_code = lane / KR * (D / 2) + 8 * (lane % KR), v_code = lane / VR * PT * (D / 2) + 4 * (lane % VR);
        const uint32_t k_pair = ((16 * (lane % KR) >> a.c.group_log2) << bl) + lane / KR,
                       v_pair = ((8 * (lane % VR) >> a.c.group_log2) << bl) + PT * (lane / VR);
        const int w0 = tile * kRows + wr;
        const int r = w0 + col;
        const bool valid = r < R.rows;
        const int t_row = R.start + (valid ? r / a.group : 0), h_row = head * a.group + (valid ? r % a.group : 0);
        const int last = valid ? R.len - R.n + r / a.group : -1;
        const int all_see = R.len - R.n + w0 / a.group;

        half8_t qf[kQInLds ? 1 : KS];
        auto q_chunk = [&](int i) {
            uint4 w = make_uint4(0, 0, 0, 0);
            if (valid) w = *reinterpret_cast<const uint4*>(a.q + t_row * a.ldq + h_row * D + 16 * i + 8 * h);
            return pairs_from_rising(w);
        };
        if constexpr (!kQInLds) {
#pragma unroll
            for (int i = 0; i < KS; ++i) qf[i] = __builtin_bit_cast(half8_t, q_chunk(i));
        }
        float16_t acc[DT];
#pragma unroll
        for (int j = 0; j < DT; ++j)
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[j][i] = 0.f;
        float m = -INFINITY, l = 0.f;

        lds_barrier();  // the last sequence's sums have been read
        if constexpr (kQInLds) {
            if (group == 0) {
#pragma unroll
                for (int i = 0; i < KS; ++i) {
                    *reinterpret_cast<uint4*>(&s.t.q[wr + col][16 * i + 8 * h]) = q_chunk(i);
                    if (i % 4 == 3) __builtin_amdgcn_sched_barrier(0);  // few registers are left
                }
            }
        }
        for (int seg = k0; seg < k1; seg += kSegment) {
            const int seg_end = min(seg + kSegment, k1);
            const int p0 = seg >> bl, pages = ((seg + (seg_end - seg + BN - 1) / BN * BN - 1) >> bl) - p0 + 1;
            lds_barrier();
            bool lost = false;
            for (int p = tid; p < pages; p += kThreads) {
                const int page = p0 + p;
                int id = -1;
                if (page < a.width && (page << bl) < k1) id = early != -2 && seg == 0 ? early : a.tables[b * a.ld_table + page];
                const bool ok = id >= 0 && id < a.c.num_blocks;
                s.run[p] = ok ? id * a.c.kv_heads + head : -1;
                lost |= !ok && (page << bl) < k1;
            }
            const bool some_lost = __syncthreads_or(lost);
            const int tiles = (seg_end - seg + BN - 1) / BN;
            // the first tile that a row of this wave does not see whole
            const int first_masked = some_lost ? 0 : max(min(all_see + 1, seg_end) - seg, 0) / BN;

            // Codes and affine pairs of a tile on their way to LDS.  A wave's chunks lie in 16
            // tokens of one block, which it looks up before the conversions of the tile
            // before and uses behind them.  (Of the nearest tile that exists: loads under a condition
            // would be waited for at its end, where their registers join those of the other way.)
            auto first_of = [&](int t) { return seg + min(max(t, 0), tiles - 1) * BN; };
            auto k_token = [&](int t, int i) { return first_of(t) + (64 * cw + kConv * i) / KR; };
            auto v_token = [&](int t) { return first_of(t) + PT * (64 / VR) * cw; };
            auto look = [&](int token) { return s.run[(token >> bl) - p0]; };
            auto in_block = [&](int token) { return static_cast<uint32_t>(token & ((1 << bl) - 1)); };
            const int codes_log2 = bl + __builtin_ctz(D / 2), pairs_log2 = bl + groups_log2 + 2;  // bytes of a block's head
            typedef uint32_t pairs_t __attribute__((ext_vector_type(PT)));
            uint32_t kc[2 * KC] = {}, ka[KC] = {}, vc[PT] = {};
            pairs_t va = {};
            int next_k[KC], next_v;
            int v_left = 0;  // tokens from a wave's first one of the values on that are there
            auto look_up = [&](int tv, int tk) {
                next_v = look(v_token(tv));
#pragma unroll
                for (int i = 0; i < KC; ++i) next_k[i] = look(k_token(tk, i));
            };
            // In two steps: where they are, and their loads.
            const uint8_t *k_from[KC], *v_from;
            const char *k_pairs_from[KC], *v_pairs_from;
            uint32_t k_off[KC], v_off;
            int left = 0;
            auto place_k = [&](int t) {
#pragma unroll
                for (int i = 0; i < KC; ++i) {
                    const int64_t run = max(__builtin_amdgcn_readfirstlane(next_k[i]), 0);
                    k_off[i] = in_block(k_token(t, i));
                    k_from[i] = a.c.k + (run << codes_log2);
                    k_pairs_from[i] = reinterpret_cast<const char*>(a.c.k_affine) + (run << pairs_log2);
                }
            };
            auto load_k = [&] {
#pragma unroll
                for (int i = 0; i < KC; ++i) {
                    const uint64_t c = load_from<uint64_t>(k_from[i], k_code + k_off[i] * (D / 2));
                    kc[2 * i] = static_cast<uint32_t>(c);
                    kc[2 * i + 1] = static_cast<uint32_t>(c >> 32);
                    ka[i] = load_from<uint32_t>(k_pairs_from[i], 4 * (k_pair + k_off[i]));
                }
            };
            auto place_v = [&](int t) {
                const int found = __builtin_amdgcn_readfirstlane(next_v);
                const int64_t run = max(found, 0);
                v_off = in_block(v_token(t));
                left = found < 0 ? 0 : k1 - v_token(t);
                v_from = a.c.v + (run << codes_log2);
                v_pairs_from = reinterpret_cast<const char*>(a.c.v_affine) + (run << pairs_log2);
            };
            auto load_v = [&] {
                v_left = left;
#pragma unroll
                for (int j = 0; j < PT; ++j) vc[j] = load_from<uint32_t>(v_from + j * (D / 2), v_code + v_off * (D / 2));
                va = load_from<pairs_t>(v_pairs_from, 4 * (v_pair + v_off));
            };
            // (tiles that do not exist go into the buffer of the one before the last, or of the
            // first ones before they are written)
            auto store_k = [&](int t) {
#pragma unroll
                for (int e = 0; e < 2 * KC; ++e) {
                    const int i = e / 2;
                    uint4* p = reinterpret_cast<uint4*>(&s.t.k[t & 1][kConv / KR * i + ct / KR][16 * (ct % KR)]);
                    p[e % 2] = elements8(nib, kc[e], ka[i]);
                }
            };
            auto store_v = [&](int t) {
                const int first = PT * (ct / VR), quad = first / 4;
                // what lies behind the last token, or in a lost block, may be no number
#pragma unroll
                for (int j = 0; j < PT; ++j) va[j] = PT * (lane / VR) + j < v_left ? va[j] : 0u;
                uint32_t f[PT / 2][8];
#pragma unroll
                for (int k = 0; k < PT / 2; ++k) {
                    const half2_t sc = scales2(va[2 * k], va[2 * k + 1]), bi = biases2(va[2 * k], va[2 * k + 1]);
                    token_pairs(nib, vc[2 * k], vc[2 * k + 1], sc, bi, 0, f[k]);
                    token_pairs(nib, vc[2 * k], vc[2 * k + 1], sc, bi, 1, f[k] + 4);
                }
                // channel ch + j lies j rows behind, its chunks exchanged as v_place does
                const int ch = 8 * (ct % VR);
                uint32_t at = 2 * BN * ch + 16 * v_place(ch, 2 * (quad / 4) + (quad & 1)) + 8 * ((quad >> 1) & 1) + 2 * (first % 4);
                asm volatile("" : "+v"(at));  // one register, not eight of them kept for the loop
                char* rows = reinterpret_cast<char*>(s.t.v[t & 1]);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    char* p = rows + (at ^ 16 * v_place(j, 0)) + 2 * BN * j;
                    if constexpr (PT == 4) *reinterpret_cast<uint2*>(p) = make_uint2(f[0][j], f[PT / 2 - 1][j]);
                    else *reinterpret_cast<uint32_t*>(p) = f[0][j];
                }
            };
            float16_t x[ST] = {};  // scores of this wave's tile, and its weights
            half8_t pf[U];
            // A tile's matrix instructions in order: PV of its values, then QK of the next one's
            // keys.  Their fragments (and those of q, where it is in LDS) are read AHEAD of them.
            constexpr int AHEAD = D == 256 ? 3 : 8, FQ = AHEAD / ST, PV = U * DT, QK = KS * ST;
            half8_t fr[AHEAD], fq[kQInLds ? FQ : 1];
            uint32_t v_read = 0;  // bytes of channel col's tokens 8h on in V^T
            auto fetch = [&](int n, int tv, int tk) {
                half8_t& f = fr[n % AHEAD];
                if (n < PV) {
                    const int u = n / DT, i = n % DT;
                    f = *reinterpret_cast<const half8_t*>(reinterpret_cast<const char*>(s.t.v[tv & 1]) +
                                                          (v_read ^ 16 * v_place(32 * i, 2 * u)) + 64 * BN * i);
                } else if (n < PV + QK) {
                    const int i = (n - PV) / ST, j = (n - PV) % ST;
                    f = *reinterpret_cast<const half8_t*>(&s.t.k[tk & 1][32 * j + col][16 * i + 8 * h]);
                }
                if constexpr (kQInLds) {
                    const int i = (n - PV) / ST;
                    if (n >= PV && n < PV + QK && (n - PV) % ST == 0) fq[i % FQ] = *reinterpret_cast<const half8_t*>(&s.t.q[wr + col][16 * i + 8 * h]);
                }
            };
            auto multiply = [&](int n) {
                const half8_t f = fr[n % AHEAD];
                if (n < PV) {
                    acc[n % DT] = __builtin_amdgcn_mfma_f32_32x32x16_f16(f, pf[n / DT], acc[n % DT], 0, 0, 0);
                } else {
                    const int i = (n - PV) / ST, j = (n - PV) % ST;
                    const half8_t q = kQInLds ? fq[kQInLds ? i % FQ : 0] : qf[kQInLds ? 0 : i];
                    if (i == 0) {
#pragma unroll
                        for (int g = 0; g < 16; ++g) x[j][g] = 0.f;
                    }
                    x[j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(f, q, x[j], 0, 0, 0);
                }
            };
            // Instructions [from, PV + QK) one after the other.
            auto multiply_from = [&](int from, int tv, int tk, auto between) {
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int n = from; n < from + AHEAD; ++n) fetch(n, tv, tk);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int n = from; n < PV + QK; ++n) {
                    multiply(n);
                    fetch(n + AHEAD, tv, tk);
                    between(n);
                    __builtin_amdgcn_sched_barrier(0);
                }
            };
            // The products of tile tv's values, then the scores of tile tk (of whatever lies
            // there behind the last one).  Beside them the scalar unit finds where the codes of
            // tiles lv and lk are.
            auto matrices = [&](int tv, int tk, int lv, int lk) {
                v_read = 2 * BN * col + 16 * v_place(col, h);
                asm volatile("" : "+v"(v_read));  // one register, not one for each place kept for the loop
                look_up(lv, lk);
                multiply_from(0, tv, tk, [&](int n) {
                    if (n == 2) place_v(lv);
                    if (n == 6) place_k(lk);
                });
            };
            // Codes that are there become tile tv's values and tile tk's keys; the next ones
            // are on their way.
            auto convert = [&](int tv, int tk) {
                store_v(tv);
                load_v();
                store_k(tk);
                load_k();
            };
            // The scores of the first tile alone.
            auto scores = [&](int t) { multiply_from(PV, t, t, [](int) {}); };
            // The weights of tile t, none where there is no such tile or its tokens are not seen.
            auto softmax = [&](int t) {
                if (__builtin_expect(t >= first_masked, 0)) {
                    const int base = seg + t * BN, most = min(last, seg_end - 1) - base - 4 * h;
#pragma unroll
                    for (int i = 0; i < ST; ++i)
#pragma unroll
                        for (int j = 0; j < 16; ++j) x[i][j] = 32 * i + 8 * (j / 4) + j % 4 > most ? -INFINITY : x[i][j];
                    if (some_lost && t < tiles) {  // a block outside the cache has no weight
#pragma unroll
                        for (int u = 0; u < U; ++u) {
                            const bool none = look(base + 16 * u) < 0;
#pragma unroll
                            for (int j = 0; j < 8; ++j) x[u / 2][8 * (u & 1) + j] = none ? -INFINITY : x[u / 2][8 * (u & 1) + j];
                        }
                    }
                }
                float mq[U];
#pragma unroll
                for (int u = 0; u < U; ++u) {  // chains side by side: one would wait for itself
                    mq[u] = x[u / 2][8 * (u & 1)];
#pragma unroll
                    for (int j = 1; j < 8; ++j) mq[u] = fmaxf(mq[u], x[u / 2][8 * (u & 1) + j]);
                }
                float mx = mq[0];
#pragma unroll
                for (int u = 1; u < U; ++u) mx = fmaxf(mx, mq[u]);
                {
                    float p = mx, q = mx;
                    swap32(p, q);
                    mx = fmaxf(p, q) * a.scale_log2;
                }
                if (__builtin_expect(__any(mx - m > kMost), 0)) {  // as in RowTile4
                    const float m_new = fmaxf(m, mx - kSet);
                    const float alpha = __builtin_amdgcn_exp2f(m - (m_new == -INFINITY ? 0.f : m_new));
                    l *= alpha;
#pragma unroll
                    for (int i = 0; i < DT; ++i) acc[i] *= alpha;
                    m = m_new;
                }
                const float ref = m == -INFINITY ? 0.f : m;
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    float p[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        p[i] = __builtin_amdgcn_exp2f(fmaf(x[u / 2][8 * (u & 1) + i], a.scale_log2, -ref));
                        pf[u][i] = static_cast<half_t>(p[i]);
                    }
                    l += ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
                }
            };

            // The next slot begins; no instruction of one moves into the other (the compiler moves
            // vector work across the barrier, into the time of the matrix cores: 169 us for 159).
            auto next_slot = [&] {
                __builtin_amdgcn_sched_barrier(0);
                lds_barrier();
                __builtin_amdgcn_sched_barrier(0);
            };
            // What a slot reads was written a slot before at the latest, into the buffer
            // that was read for the last time a slot before that.  Both groups go through as
            // many slots, one apart.  (Tiles that do not exist are the last one again: finite
            // values, no weights.)
            auto codes_of = [&](int tv, int tk) {
                look_up(tv, tk);
                place_v(tv);
                place_k(tk);
            };
            const int first = SPLIT == 1 ? 0 : group;
            codes_of(first, first);
            load_v();
            load_k();
            codes_of(first + SPLIT, first + SPLIT);
            convert(first, first);
            codes_of(first + 2 * SPLIT, first + 2 * SPLIT);
            lds_barrier();
            scores(first);
            if constexpr (SPLIT == 2) lds_barrier();
            store_k(first + SPLIT);
            load_k();
            softmax(first);
            lds_barrier();
            if (group == 1) {
                if constexpr (SPLIT == 1) {
                    look_up(2, 3);
                    place_k(3);
                    convert(1, 2);
                }
                lds_barrier();
            }
            if constexpr (SPLIT == 1) {
                // tile j: slot 2j of the first group, 2j + 1 of the second
                for (int j = 0; j < tiles; ++j) {
                    matrices(j, j + 1, j + 2 + group, j + 3 + group);
                    next_slot();
                    convert(j + 1 + group, j + 2 + group);
                    softmax(j + 1);
                    next_slot();
                }
            } else {
                // tile t: slot t of group t % 2
                for (int t = group; t < (tiles + 1) / 2 * 2; t += 2) {
                    matrices(t, t + 2, t + 4, t + 6);
                    next_slot();
                    convert(t + 2, t + 4);
                    softmax(t + 2);
                    next_slot();
                }
            }
            if (group == 0) lds_barrier();
        }
        {
            float p = l, q = l;
            swap32(p, q);
            l = p + q;
        }
        float f0 = 1.f, f1 = 0.f;
        if constexpr (SPLIT == 2) {
            lds_barrier();  // the tiles and q have been read
            if (group == 1) {
#pragma unroll
                for (int j = 0; j < DT; ++j)
#pragma unroll
                    for (int i = 0; i < 16; i += 4)
                        *reinterpret_cast<float4_t*>(&s.sum.o[wr + col][32 * j + 2 * i + 4 * h]) =
                            float4_t{acc[j][i], acc[j][i + 1], acc[j][i + 2], acc[j][i + 3]};
                if (h == 0) {
                    s.sum.m[wr + col] = m;
                    s.sum.l[wr + col] = l;
                }
            }
            lds_barrier();
            if (group == 1) return;
            const float m1 = s.sum.m[wr + col], top = fmaxf(m, m1), ref = top == -INFINITY ? 0.f : top;
            f0 = __builtin_amdgcn_exp2f(m - ref);
            f1 = __builtin_amdgcn_exp2f(m1 - ref);
            m = top;
            l = l * f0 + s.sum.l[wr + col] * f1;
        }
        if (!valid) return;
        auto sum4 = [&](int j, int i) {
            float4_t o = {acc[j][i], acc[j][i + 1], acc[j][i + 2], acc[j][i + 3]};
            if constexpr (SPLIT == 2) o = o * f0 + *reinterpret_cast<const float4_t*>(&s.sum.o[wr + col][32 * j + 2 * i + 4 * h]) * f1;
            return o;
        };
        if (slot < 0) {
            const float inv = inverse(l);
            int row = w0 + col;
            asm volatile("" : "+v"(row));  // divided again: the quotients are not kept over the loop
            uint16_t* to = a.o + (R.start + row / a.group) * a.ldo + (head * a.group + row % a.group) * D;
#pragma unroll
            for (int j = 0; j < DT; ++j)
#pragma unroll
                for (int i = 0; i < 16; i += 4) {
                    const float4_t o = sum4(j, i);
                    uint2 w;
                    w.x = pack_h2(static_cast<half_t>(o[0] * inv), static_cast<half_t>(o[1] * inv));
                    w.y = pack_h2(static_cast<half_t>(o[2] * inv), static_cast<half_t>(o[3] * inv));
                    *reinterpret_cast<uint2*>(to + 32 * j + 2 * i + 4 * h) = w;
                }
        } else {
            const int64_t row = static_cast<int64_t>(slot) * kRows + wr + col;
#pragma unroll
            for (int j = 0; j < DT; ++j)
#pragma unroll
                for (int i = 0; i < 16; i += 4)
                    *reinterpret_cast<float4_t*>(a.part_o + row * D + 32 * j + 2 * i + 4 * h) = sum4(j, i);
            if (h == 0) a.part_ml[row] = make_float2(m, l);
        }
    }
};

template <int D>
int launch_attend4(Args4 a, const Plan& p, int64_t blocks, int64_t max_rows, char* workspace, hipStream_t s) {
    const char* where = "kv4_attention launch";
    const int zero_other = a.zero_other;
    a.zero_other = p.few.on ? zero_other : 0;
    const int64_t few_rows = p.many.on ? kFewRows : max_rows;
    auto few = [&](auto tile) { return launch_part<RowTile4<D, 8>, decltype(tile)>(a, p.few, blocks, few_rows, workspace, s, where); };
    int rc = GDSLLM_OK;
    if constexpr (D == 256) {
        // One workgroup to a compute unit.  Eight waves for the bytes under way; four, whose sums meet
        // sooner, where tiles are full and a workgroup has few tokens.  (2 key heads of 16 query heads
        // each, four waves and eight: 32 requests of up to 2000 tokens 22.1 us and 23.0, 4000 22.7 and 23.5,
        // 8000 31.1 and 31.0, 16000 51.5 and 45.5; one of 60000 25.2 and 26.4, 80000 24.3 and 24.1, 100000 31.1
        // and 30.2, 160000 37.3 and 33.6.  Of several the longest says about twice what they have.  Half full,
        // 4 requests over 4 key heads of 8, up to 4000 20.7 and 19.8, 16000 22.3 and 21.7.)
        const int64_t most = (a.requests > 1 ? 1024 : 640) * static_cast<int64_t>(p.few.groups);
        if (few_rows >= 16 && p.few.sequences * p.few.longest < most) rc = few(RowTile4<D, 4>{});
        else rc = few(RowTile4<D, 8>{});
    } else {
        rc = few(RowTile4<D, 4>{});
    }
    if (rc) return rc;
    a.zero_other = p.few.on ? 0 : zero_other;
    char* ws = workspace + p.few.bytes;
    if constexpr (D <= 128)
        if (p.many.rows == 256) return launch_part<PromptTile4<D, 1>, PromptTile4<D, 1>>(a, p.many, blocks, max_rows, ws, s, where);
    return launch_part<PromptTile4<D, 2>, PromptTile4<D, 2>>(a, p.many, blocks, max_rows, ws, s, where);
}

}  // namespace
}  // namespace gdsllm

using namespace gdsllm;

extern "C" size_t gdsllm_kv4_attention_workspace_size(int64_t requests, int64_t q_heads, int64_t kv_heads, int64_t head_dim,
                                                      int64_t max_new, int64_t max_len) {
    if (!attend_sizes(requests, q_heads, kv_heads, head_dim, max_new, max_len)) return 0;
    return workspace_bound(requests, q_heads, kv_heads, head_dim, max_new, max_len, {kPromptsPerCu, true});
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
                             starts, requests, scale, max_new, max_len, zero_other, workspace, workspace_bytes,
                             {kPromptsPerCu, true}, a, &c))
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
