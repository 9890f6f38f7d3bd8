// Attention over the 8-bit KV cache (kv_cache.hip writes it).
//
// For query row t of request b (n_b rows in this call, len_b tokens held) and
// query head h of kv head h / G:
//   x_j = scale * k_scale * (q . code_j),  j <= len_b - n_b + t
//   o   = sum_j 2^(x_j log2 e) v_j / sum_j 2^(x_j log2 e)
// in one pass over the tokens with a running reference m.  Codes enter the matrix
// cores as the fp16 values they are, so the products q . code and P . code are
// exact and summed in fp32; the scales stay outside: a block's key scale
// multiplies its scores, and its value scale is carried in the exponent.  With
// e = log2(v_scale) and m 7 to 11 below the largest y_j = x_j log2 e + e so far,
//   acc += 2^(y_j - m) * code_j,   l += 2^(y_j - m) / v_scale,   o = acc / l.
// The weights are rounded to fp16 for the product with the codes (the matrix cores
// take no wider operand at this rate) and for it alone: l takes them in fp32,
// since in a block of small values they may be less than fp16 holds.  That
// rounding, the one before the last, is half an fp16 step of a weight, and 2^-25
// at least: the largest is 2^7 to 2^11, so a key's share of the values is off by
// 2^-11 of itself or 2^-32 of the largest share, whichever is more.
//
// The G query heads of a kv head and the query rows share its keys: they are
// the columns of a matrix tile (row r = token r / G, head r % G), 16 of them for
// requests of up to 32 rows (RowTile), 128 or 256 for prompts (PromptTile).
//  * Decode reads each code once and is bound by that: 32 requests of 8192 tokens
//    over 8 heads 273 MB in 59 us, 4.6 TB/s, 53 us of it attend_shared (a large
//    copy reaches 4.75); one of 131072 tokens over 2 heads of 256 134 MB in 37 us,
//    30 of them attend_shared.  A short sequence (777 tokens, 32 heads, 9.6 us) is
//    one chain of memory latencies: a launch, its length and table, its scales,
//    then three tiles of codes to a wave.
//  * Prompts are bound by vector work beside the matrix cores (by counters, softmax
//    and the codes' conversion take 40% of a SIMD's cycles, its matrix core 35%):
//    4096 tokens of 32 heads 174 us, 790 TFLOP/s of a large product's 1060; 4 chunks
//    of 300 tokens with up to 5000 held 160 us, 515 TFLOP/s: 448 tiles of unequal
//    length are 1.75 to a compute unit.  Even shares of their keys take 257 us, 92 of
//    them in attend_join, which gives each of 57000 rows, most of two parts,
//    a workgroup of its own; 16 such chunks reach 674.

#include "kv_attend.h"
#include "kv_cache.h"

namespace gdsllm {
namespace {

typedef AttendArgs<KvCache> Args8;
// Workgroups of PromptTile that a compute unit holds at once.
constexpr int prompts_per_cu(int64_t D) { return D == 256 ? 1 : 2; }

// 16 rows over blocks [block0, block1) of a sequence, by NW waves.  Matrix tiles
// are 16x16x32 and nothing passes through LDS but the block table and the waves'
// sums:
//  * scores S^T = K Q^T: lane l gives key row l % 16 and 16 of each 64 channels
//    (one 16-byte load; Q's operand takes the same order), and receives, for
//    query l % 16, tokens 4 * group .. + 3 of each 16;
//  * O^T = V^T P^T: its B operand is exactly those eight weights of two score
//    tiles, in place; V's operand needs eight tokens of one channel in a lane:
//    lanes load D/16 channels of the eight tokens and transpose 4x4 bytes with
//    v_perm.
template <bool E4M3, int D, int NW_>
struct RowTile {
    typedef Args8 Args;
    static constexpr int kRows = 16, kD = D, kPerCu = per_cu(D), kBegin = 0;
    static constexpr bool kRowJoin = false;
    static constexpr int kThreads = NW_ * 64;
    static constexpr int NT = 2;        // score tiles of an iteration
    static constexpr int NW = NW_;
    static constexpr int KS = D / 32;   // score steps of 32 channels
    static constexpr int DB = D / 16;   // channels of V a lane holds
    static constexpr int VW = DB / 4;   // the same in dwords
    static constexpr int TT = 16 * NT;  // tokens of an iteration
    struct Codes {
        uint32_t k[NT][D / 16];
        uint32_t v[NT][4][VW];
    };
    struct Lds {
        int id[kMaxPages];
        float c[kMaxPages], e[kMaxPages], inv[kMaxPages];
        float m[NW][16], l[NW][16];
        float o[NW][16][D + 4];
    };

    // Codes of 16 tokens from `kb` (`vb`) on, wave-uniform, into slot t.
    __device__ __forceinline__ static void load_k(Codes& w, int t, const uint8_t* kb, uint32_t klane) {
#pragma unroll
        for (int i = 0; i < D / 64; ++i) {
            const u32x4_t x = __builtin_nontemporal_load(reinterpret_cast<const u32x4_t*>(kb + klane + 64 * i));
#pragma unroll
            for (int j = 0; j < 4; ++j) w.k[t][4 * i + j] = x[j];
        }
    }
    __device__ __forceinline__ static void load_v(Codes& w, int t, const uint8_t* vb, uint32_t vlane) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint8_t* p = vb + vlane + i * D;
            if constexpr (VW == 1) {
                w.v[t][i][0] = __builtin_nontemporal_load(reinterpret_cast<const uint32_t*>(p));
            } else if constexpr (VW == 2) {
                const uint64_t x = __builtin_nontemporal_load(reinterpret_cast<const uint64_t*>(p));
                w.v[t][i][0] = static_cast<uint32_t>(x);
                w.v[t][i][1] = static_cast<uint32_t>(x >> 32);
            } else {
                const u32x4_t x = __builtin_nontemporal_load(reinterpret_cast<const u32x4_t*>(p));
#pragma unroll
                for (int j = 0; j < 4; ++j) w.v[t][i][j] = x[j];
            }
        }
    }

    // `slot` < 0: the sequence is whole, its rows are written to o; else its sums
    // go to that part.  `early`: entry threadIdx.x of the request's block table,
    // loaded ahead of its length (only where block0 is 0 and a thread has each
    // entry of a segment), else -2.
    __device__ static void run(const Args& a, Lds& s, int b, const Rows<16>& R, int tile, int head, int block0,
                               int block1, int slot, int early) {
        const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), col = lane & 15,
                  g = lane >> 4;
        const int bl = a.c.block_log2;
        const uint32_t klane = col * D + 16 * g, vlane = 4 * g * D + col * DB;
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
            if (valid) w = *reinterpret_cast<const uint4*>(a.q + t_row * a.ldq + h_row * D + 64 * (i / 2) + 16 * g + 8 * (i & 1));
            qf[i] = __builtin_bit_cast(half8_t, w);
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
                s.inv[p] = ok ? 1.f : 0.f;
                lost |= !ok && (page << bl) < k1;
            }
            const bool some_lost = __syncthreads_or(lost);
            auto row_of = [&](int token) {
                const int id = __builtin_amdgcn_readfirstlane(s.id[(token >> bl) - p0]);
                return (((static_cast<int64_t>(id) * a.c.kv_heads + head) << bl) + (token & ((1 << bl) - 1))) * D;
            };
            constexpr int step = NW * TT;
            int base = seg + wave * TT;
            // the scales, and behind them the first codes
            float ks = 0.f, vs = 0.f;
            int64_t sc = 0;
            if (tid < pages) {
                sc = static_cast<int64_t>(s.id[tid]) * a.c.kv_heads + head;
                ks = a.c.k_scale[sc];
                vs = a.c.v_scale[sc];
            }
            Codes w;
            if (base < seg_end) {
#pragma unroll
                for (int t = 0; t < NT; ++t) load_k(w, t, a.c.k + row_of(base + 16 * t), klane);
#pragma unroll
                for (int t = 0; t < NT; ++t) load_v(w, t, a.c.v + row_of(base + 16 * t), vlane);
            }
            for (int p = tid; p < pages; p += NW * 64) {
                if (p != tid) {
                    sc = static_cast<int64_t>(s.id[p]) * a.c.kv_heads + head;
                    ks = a.c.k_scale[sc];
                    vs = a.c.v_scale[sc];
                }
                vs = fmaxf(vs, 0x1p-64f);
                s.c[p] = ks * a.scale_log2;
                s.e[p] = log2f(vs);
                s.inv[p] = s.inv[p] / vs;
            }
            lds_barrier();
            for (; base < seg_end; base += step) {
                const bool more = base + step < seg_end;
                float x[NT][4];
                float mx = -INFINITY;
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    float4_t sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int i = 0; i < KS; ++i) {
                        uint32_t f[4];
                        codes_to_f16<E4M3>(w.k[t][2 * i], f[0], f[1]);
                        codes_to_f16<E4M3>(w.k[t][2 * i + 1], f[2], f[3]);
                        const half8_t kf = __builtin_bit_cast(half8_t, make_uint4(f[0], f[1], f[2], f[3]));
                        sum = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, qf[i], sum, 0, 0, 0);
                    }
                    const int p = ((base + 16 * t) >> bl) - p0;
                    const float c = s.c[p], e = s.e[p];
#pragma unroll
                    for (int i = 0; i < 4; ++i) x[t][i] = fmaf(sum[i], c, e);
                }
                if (more) {  // the keys' registers are free: the next tile's
#pragma unroll
                    for (int t = 0; t < NT; ++t) load_k(w, t, a.c.k + row_of(base + step + 16 * t), klane);
                }
                if (base + TT - 1 > all_see || base + TT > k1 || some_lost) {
#pragma unroll
                    for (int t = 0; t < NT; ++t) {
                        // a block outside the cache has no weight
                        const bool none = s.inv[((base + 16 * t) >> bl) - p0] == 0.f;
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const int j = base + 16 * t + 4 * g + i;
                            if (j > last || j >= k1 || none) x[t][i] = -INFINITY;
                            if (j >= k1 || none) {  // what lies there may be no number
#pragma unroll
                                for (int u = 0; u < VW; ++u) w.v[t][i][u] = 0;
                            }
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
                for (int t = 0; t < NT; ++t) {
                    const float inv = s.inv[((base + 16 * t) >> bl) - p0];
                    float sum = 0.f;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float p = __builtin_amdgcn_exp2f(x[t][i] - ref);
                        sum += p;
                        pf[t / 2][4 * (t & 1) + i] = static_cast<half_t>(p);
                    }
                    l = fmaf(sum, inv, l);
                }
#pragma unroll
                for (int u = 0; u < NT / 2; ++u)
#pragma unroll
                    for (int c = 0; c < VW; ++c) {
                        uint32_t f[4][4];  // [channel][token pair]
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            const uint32_t t0 = w.v[2 * u + k / 2][2 * (k & 1)][c], t1 = w.v[2 * u + k / 2][2 * (k & 1) + 1][c];
                            codes_to_f16<E4M3>(__builtin_amdgcn_perm(t1, t0, 0x05010400u), f[0][k], f[1][k]);
                            codes_to_f16<E4M3>(__builtin_amdgcn_perm(t1, t0, 0x07030602u), f[2][k], f[3][k]);
                        }
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const half8_t vf = __builtin_bit_cast(half8_t, make_uint4(f[j][0], f[j][1], f[j][2], f[j][3]));
                            acc[4 * c + j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, pf[u], acc[4 * c + j], 0, 0, 0);
                        }
                    }
                if (more) {
#pragma unroll
                    for (int t = 0; t < NT; ++t) load_v(w, t, a.c.v + row_of(base + step + 16 * t), vlane);
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
// prompts.  BN tokens at a time are converted to fp16 once, into LDS
// (two buffers, one barrier a tile), while the tile before is worked on; matrix
// tiles are 32x32x16:
//  * S^T = K Q^T: K [token][channel] from LDS, Q in registers; lane l receives,
//    for query l % 32, tokens 8b + 4h + j of each 32 (h = l / 32);
//  * O^T = V^T P^T: again those weights are the B operand in place, eight tokens
//    16u + 8(i/4) + 4h + i%4 to a lane, and V lies in LDS transposed, [channel]
//    [token], with its tokens in that order, so its operand is one 16-byte read.
// The four-token pieces of V^T come from 4x4 byte transposes of the codes.  Rows
// of both tiles are 16 bytes longer than their data: reads and writes touch
// every bank once.
template <bool E4M3, int D, int NW>
struct PromptTile {
    typedef Args8 Args;
    static constexpr int kRows = 32 * NW, kThreads = 64 * NW, kD = D, kPerCu = prompts_per_cu(D), kBegin = 0;
    static constexpr bool kRowJoin = false;
    static constexpr int BN = D == 256 ? 32 : 64;
    static constexpr int ST = BN / 32, KS = D / 16, DT = D / 32, U = BN / 16;
    // 16-code chunks of K, and the ones a thread converts (the last threads none where there are fewer)
    static constexpr int KT = BN * D / 16, KC = (KT + kThreads - 1) / kThreads;
    // (four tokens, 8 channels) pieces of V, and the ones a thread converts
    static constexpr int VQ = BN / 4, VC = VQ * (D / 8), VN = (VC + kThreads - 1) / kThreads;
    struct Page {
        float c, e, inv;
        int id;
    };
    struct Lds {
        Page page[kMaxPages];
        uint16_t k[2][BN][D + 8];
        uint16_t v[2][D][BN + 8];
    };
    struct Codes {
        u32x4_t k[KC];
        uint64_t v[VN][4];
    };

    __device__ static void run(const Args& a, Lds& s, int b, const Rows<kRows>& R, int tile, int head, int block0,
                               int block1, int slot, int early) {
        const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), col = lane & 31,
                  h = lane >> 5;
        const int bl = a.c.block_log2;
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
            qf[i] = __builtin_bit_cast(half8_t, w);
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
                const int64_t sc = static_cast<int64_t>(ok ? id : 0) * a.c.kv_heads + head;
                const float vs = fmaxf(a.c.v_scale[sc], 0x1p-64f);
                s.page[p] = {fmaxf(a.c.k_scale[sc], 0x1p-64f) * a.scale_log2, log2f(vs), ok ? 1.f / vs : 0.f, ok ? id : 0};
                lost |= !ok && (page << bl) < k1;
            }
            const bool some_lost = __syncthreads_or(lost);

            auto load = [&](Codes& w, int base) {
#pragma unroll
                for (int i = 0; i < KC; ++i) {
                    const int c = tid + kThreads * i, token = base + c / (D / 16);
                    if (KT % kThreads != 0 && c >= KT) continue;
                    const int64_t row = ((static_cast<int64_t>(s.page[(token >> bl) - p0].id) * a.c.kv_heads + head) << bl) +
                                        (token & ((1 << bl) - 1));
                    w.k[i] = *reinterpret_cast<const u32x4_t*>(a.c.k + row * D + 16 * (c % (D / 16)));
                }
#pragma unroll
                for (int i = 0; i < VN; ++i) {
                    const int c = tid + kThreads * i, token = base + 4 * (c % VQ);
                    if (VC % kThreads == 0 || c < VC) {
                        const int64_t row = ((static_cast<int64_t>(s.page[(token >> bl) - p0].id) * a.c.kv_heads + head) << bl) +
                                            (token & ((1 << bl) - 1));
                        const uint8_t* p = a.c.v + row * D + 8 * (c / VQ);
#pragma unroll
                        for (int j = 0; j < 4; ++j) w.v[i][j] = *reinterpret_cast<const uint64_t*>(p + j * D);
                    }
                }
            };
            auto store = [&](Codes& w, int base, int buf) {
#pragma unroll
                for (int i = 0; i < KC; ++i) {
                    const int c = tid + kThreads * i;
                    if (KT % kThreads != 0 && c >= KT) continue;
                    uint32_t f[8];
#pragma unroll
                    for (int j = 0; j < 4; ++j) codes_to_f16<E4M3>(w.k[i][j], f[2 * j], f[2 * j + 1]);
                    uint4* p = reinterpret_cast<uint4*>(&s.k[buf][c / (D / 16)][16 * (c % (D / 16))]);
                    p[0] = make_uint4(f[0], f[1], f[2], f[3]);
                    p[1] = make_uint4(f[4], f[5], f[6], f[7]);
                }
                const bool tail = base + BN > k1 || some_lost;
#pragma unroll
                for (int i = 0; i < VN; ++i) {
                    const int c = tid + kThreads * i, quad = c % VQ;
                    if (VC % kThreads == 0 || c < VC) {
                        if (tail) {  // what lies behind the last token, or in a lost block, may be no number
                            const int token = base + 4 * quad;
                            const bool none = s.page[(token >> bl) - p0].inv == 0.f;
#pragma unroll
                            for (int j = 0; j < 4; ++j)
                                if (none || token + j >= k1) w.v[i][j] = 0;
                        }
                        const int pos = 16 * (quad / 4) + 8 * (quad & 1) + 4 * ((quad >> 1) & 1);
#pragma unroll
                        for (int x = 0; x < 2; ++x) {
                            uint32_t t[4], f[4][2];
#pragma unroll
                            for (int j = 0; j < 4; ++j) t[j] = static_cast<uint32_t>(w.v[i][j] >> (32 * x));
#pragma unroll
                            for (int k = 0; k < 2; ++k) {
                                codes_to_f16<E4M3>(__builtin_amdgcn_perm(t[2 * k + 1], t[2 * k], 0x05010400u), f[0][k], f[1][k]);
                                codes_to_f16<E4M3>(__builtin_amdgcn_perm(t[2 * k + 1], t[2 * k], 0x07030602u), f[2][k], f[3][k]);
                            }
#pragma unroll
                            for (int j = 0; j < 4; ++j)
                                *reinterpret_cast<uint2*>(&s.v[buf][8 * (c / VQ) + 4 * x + j][pos]) = make_uint2(f[j][0], f[j][1]);
                        }
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
                                if (j > last || j >= k1 || (some_lost && s.page[(j >> bl) - p0].inv == 0.f)) x[t][i] = -INFINITY;
                            }
                    }
                    Page pg[U];
                    float mx = -INFINITY;
#pragma unroll
                    for (int u = 0; u < U; ++u) {
                        pg[u] = s.page[((base + 16 * u) >> bl) - p0];
                        const float16_t& y = x[u / 2];
                        const int o = 8 * (u & 1);
                        const float g = fmaxf(fmaxf(fmaxf(y[o], y[o + 1]), fmaxf(y[o + 2], y[o + 3])),
                                              fmaxf(fmaxf(y[o + 4], y[o + 5]), fmaxf(y[o + 6], y[o + 7])));
                        mx = fmaxf(mx, fmaf(g, pg[u].c, pg[u].e));
                    }
                    {
                        float p = mx, q = mx;
                        swap32(p, q);
                        mx = fmaxf(p, q);
                    }
                    if (__any(mx - m > kMost)) {  // as in RowTile
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
                        const float er = pg[u].e - ref;
                        half8_t pf;
                        // the sum takes the weights before they are rounded: a block of small
                        // values has weights that fp16 does not hold, 1 / v_scale times which are
                        // its share of the softmax
                        float p[8];
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            p[i] = __builtin_amdgcn_exp2f(fmaf(x[u / 2][8 * (u & 1) + i], pg[u].c, er));
                            pf[i] = static_cast<half_t>(p[i]);
                        }
                        l = fmaf(((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7])), pg[u].inv, l);
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

template <bool E4M3, int D>
int launch_attend(Args8 a, const Plan& p, int64_t blocks, int64_t max_rows, char* workspace, hipStream_t s) {
    const int zero_other = a.zero_other;
    a.zero_other = p.few.on ? zero_other : 0;
    if (int rc = launch_part<RowTile<E4M3, D, 8>, RowTile<E4M3, D, 4>>(a, p.few, blocks, p.many.on ? kFewRows : max_rows, workspace, s, "kv_attention launch"))
        return rc;
    a.zero_other = p.few.on ? 0 : zero_other;
    char* ws = workspace + p.few.bytes;
    if constexpr (D <= 128)
        if (p.many.rows == 256) return launch_part<PromptTile<E4M3, D, 8>, PromptTile<E4M3, D, 4>>(a, p.many, blocks, max_rows, ws, s, "kv_attention launch");
    return launch_part<PromptTile<E4M3, D, 4>, PromptTile<E4M3, D, 4>>(a, p.many, blocks, max_rows, ws, s, "kv_attention launch");
}

}  // namespace
}  // namespace gdsllm

using namespace gdsllm;

extern "C" size_t gdsllm_kv_attention_workspace_size(int64_t requests, int64_t q_heads, int64_t kv_heads,
                                                     int64_t head_dim, int64_t max_new, int64_t max_len) {
    if (!attend_sizes(requests, q_heads, kv_heads, head_dim, max_new, max_len)) return 0;
    return workspace_bound(requests, q_heads, kv_heads, head_dim, max_new, max_len, {prompts_per_cu(head_dim), false});
}

extern "C" int gdsllm_kv_attention(const gdsllm_kv_cache8* cache, const void* q, int64_t ldq, void* o, int64_t ldo,
                                   int64_t tokens, int64_t q_heads, const int32_t* block_tables, int64_t table_width,
                                   int64_t ld_table, const int32_t* lens, const int32_t* starts, int64_t requests,
                                   float scale, int64_t max_new, int64_t max_len, int zero_other, void* workspace,
                                   size_t workspace_bytes, void* stream) {
    Args8 a{};
    AttendCall c;
    if (int rc = kv_cache_args(cache, "kv_attention", &a.c)) return rc;
    if (int rc = attend_call("kv_attention", cache, q, ldq, o, ldo, tokens, q_heads, block_tables, table_width, ld_table, lens,
                             starts, requests, scale, max_new, max_len, zero_other, workspace, workspace_bytes,
                             {prompts_per_cu(cache->head_dim), false}, a, &c))
        return rc;
    if (c.empty) return ok();
    const int64_t D = cache->head_dim;
    const bool e4m3 = cache->format == GDSLLM_KV_E4M3;
    const hipStream_t s = as_stream(stream);
    char* ws = static_cast<char*>(workspace);
    int rc = GDSLLM_OK;
#define GDSLLM_ATTEND(DIM)                                                          \
    if (D == DIM)                                                                   \
        rc = e4m3 ? launch_attend<true, DIM>(a, c.plan, c.blocks, c.max_rows, ws, s)           \
                  : launch_attend<false, DIM>(a, c.plan, c.blocks, c.max_rows, ws, s);
    GDSLLM_ATTEND(64)
    GDSLLM_ATTEND(128)
    GDSLLM_ATTEND(256)
#undef GDSLLM_ATTEND
    return rc ? rc : ok();
}
