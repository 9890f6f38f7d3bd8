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

#include <algorithm>
#include <climits>

#include "kv_cache.h"
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

struct AttendArgs {
    KvCache c;
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
    int zero_other;          // rows of no request are set to zero
};

// A request's rows, in tiles of RT, and the keys they may see.
template <int RT>
struct Rows {
    int start, n, len, rows;
    __device__ __forceinline__ Rows(const AttendArgs& a, int b) {
        const int s0 = a.starts[b], s1 = a.starts[b + 1], held = a.lens[b];
        start = min(max(s0, 0), a.tokens);
        n = min(max(s1 - start, 0), a.tokens - start);
        len = min(max(held, 0), a.width << a.c.block_log2);
        rows = n * a.group;
        if (rows < a.min_rows || rows > a.max_rows) rows = 0;
    }
    // Keys that the last of rows [r0, r0 + count) sees.
    __device__ __forceinline__ int keys(const AttendArgs& a, int r0, int count) const {
        const int last = (min(r0 + count, rows) - 1) / a.group;
        return max(len - n + last + 1, 0);
    }
    __device__ __forceinline__ int tiles() const { return (rows + RT - 1) / RT; }
    // Blocks of kBlock tokens to each of its sequences (row tile and kv head).
    __device__ __forceinline__ int blocks() const { return max((len + kBlock - 1) / kBlock, 1); }
    __device__ __forceinline__ int work(const AttendArgs& a) const { return min(tiles(), a.tiles) * a.c.kv_heads * blocks(); }
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

// Workgroups of attend_shared that a compute unit holds at once (registers: 16
// rows of accumulators, a tile of codes and Q grow with D).  At D = 256 one, so
// that a long sequence leaves half as many parts: 131072 tokens 36.8 us against
// 41.1 with two.
constexpr int per_cu(int64_t D) { return D == 64 ? 4 : D == 128 ? 3 : 1; }

__device__ __forceinline__ float inverse(float l) { return l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l); }

// Rows of no request: before the first one's and behind the last one's.
__device__ __forceinline__ void zero_other_rows(const AttendArgs& a, int D) {
    if (!a.zero_other) return;
    const int before = min(max(a.starts[0], 0), a.tokens), end = min(max(a.starts[a.requests], before), a.tokens);
    for (int64_t i = blockIdx.x; i < before + a.tokens - end; i += gridDim.x) {
        const int64_t t = i < before ? i : end + i - before;
        for (int c = threadIdx.x; c < a.q_heads * D / 8; c += blockDim.x)
            *reinterpret_cast<uint4*>(a.o + t * a.ldo + 8 * c) = make_uint4(0, 0, 0, 0);
    }
}

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
    static constexpr int kRows = 16, kD = D, kPerCu = per_cu(D);
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
    __device__ static void run(const AttendArgs& a, Lds& s, int b, const Rows<16>& R, int tile, int head, int block0,
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
    static constexpr int kRows = 32 * NW, kThreads = 64 * NW, kD = D, kPerCu = D == 256 ? 1 : 2;
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

    __device__ static void run(const AttendArgs& a, Lds& s, int b, const Rows<kRows>& R, int tile, int head, int block0,
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

// One workgroup to a sequence (grid: row tiles times kv heads, requests).  Later
// tiles see more keys: they are dealt first.
template <class T>
__global__ __launch_bounds__(T::kThreads) void attend_whole(AttendArgs a) {
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
// work for itself, 256 a step, and looks up where its share begins.  A sequence
// that lies in several shares leaves a part in each: a workgroup has at most
// two, the one its share begins with and the one it ends in.

template <class T>
__global__ __launch_bounds__(256, T::kPerCu) void attend_shared(AttendArgs a) {
    static_assert(T::kThreads == 256, "the sums over requests go 256 a step");
    extern __shared__ __attribute__((aligned(16))) char raw[];
    typename T::Lds& s = *reinterpret_cast<typename T::Lds*>(raw);
    __shared__ int s_part[4], s_request, s_begin;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, wg = blockIdx.x;
    zero_other_rows(a, T::kD);
    int total = 0, share = 0;
    for (int pass = 0; pass < 2; ++pass) {
        int carry = 0;
        for (int b0 = 0; b0 < a.requests; b0 += 256) {
            const int b = b0 + tid, w = b < a.requests ? Rows<T::kRows>(a, b).work(a) : 0;
            int upto = wave_scan(w);
            __syncthreads();
            if (lane == 63) s_part[wave] = upto;
            __syncthreads();
            for (int i = 0; i < wave; ++i) upto += s_part[i];
            const int begin = carry + upto - w;
            carry += s_part[0] + s_part[1] + s_part[2] + s_part[3];
            if (a.requests <= 256) {  // one step: the sum is all here
                total = carry;
                share = max((total + a.groups - 1) / a.groups, 4);
            }
            const int at = wg * share;
            if (share > 0 && w > 0 && begin <= at && at < begin + w) s_request = b, s_begin = begin;
        }
        if (a.requests <= 256) break;
        total = carry;
        share = max((total + a.groups - 1) / a.groups, 4);
    }
    __syncthreads();
    int at = wg * share, b = s_request, begin = s_begin;
    const int end = min(at + share, total);
    if (at >= end) return;
    bool first = true;
    while (at < end) {
        Rows<T::kRows> R(a, b);
        while (at >= begin + R.work(a)) {
            begin += R.work(a);
            R = Rows<T::kRows>(a, ++b);
        }
        const int blocks = R.blocks(), sequence = (at - begin) / blocks, block0 = at - begin - sequence * blocks;
        const int block1 = min(blocks, block0 + end - at);
        const int head = sequence % a.c.kv_heads, tile = sequence / a.c.kv_heads;
        const bool whole = block0 == 0 && block1 == blocks;
        const int slot = 2 * wg + (first ? 0 : 1);
        if (block0 == 0 && tid == 0)
            a.parts[(static_cast<int64_t>(b) * a.tiles + tile) * a.c.kv_heads + head] =
                make_int2(slot, whole ? 0 : 1 + (blocks - block1 + share - 1) / share);
        T::run(a, s, b, R, tile, head, block0, block1, whole ? -1 : slot, -2);
        if (block0 == 0)  // more rows than the caller said: whole, by whoever begins the tile below
            for (int t = tile + a.tiles; t < R.tiles(); t += a.tiles) T::run(a, s, b, R, t, head, 0, blocks, -1, -2);
        at += block1 - block0;
        first = false;
    }
}

// Sequences that several workgroups had a part of: one workgroup to a row (to
// every rows-th one where the caller's bound on the rows was too small) adds their
// sums.  Part 0 lies in slot `first`, part i in slot 2 * (first / 2 + i).  Its
// threads first take the parts' maxima and turn them into factors, then D/4
// threads of four channels in each of NG groups run over every NGth part, and the
// groups' sums meet in LDS in a fixed order.
template <int RT, int D, int THREADS>
__global__ __launch_bounds__(THREADS) void attend_join(AttendArgs a, int rows) {
    constexpr int TPR = D / 4, NG = THREADS / TPR, NWV = THREADS / 64, EARLY = 2;
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

// One launch of a call: the requests with min_rows to max_rows rows, in tiles of
// `rows` of them.
struct Part {
    bool on = false;
    int rows = 0, min_rows = 0, max_rows = INT_MAX, tiles = 0;
    int64_t sequences = 0;  // (request, row tile, kv head)
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
    p->groups = whole ? 0 : static_cast<int>(std::min<int64_t>(resident, p->sequences * ((max_len + 255) / 256)));
    p->sums = static_cast<size_t>(p->groups) * 2 * p->rows;
    p->bytes = part_bytes(p->groups, p->rows, p->sequences, head_dim);
}

// Workgroups that the device holds at once, of 16-row and of 128-row tiles.
int64_t resident_few(int64_t head_dim) { return per_cu(head_dim) * static_cast<int64_t>(kCus); }
int64_t resident_many(int64_t head_dim) { return (head_dim == 256 ? 1 : 2) * static_cast<int64_t>(kCus); }

// One workgroup to a sequence where none is long or there are many of them, else
// as many workgroups as the device holds at once, with even shares.  (256 requests
// of up to 4000 tokens over 8 heads: 218 us whole, 236 shared out; a prompt of 500 tokens
// behind 1500, 128 tiles: 62 whole, 66 shared out; one of 64 in 32 tiles: 57 and 34.)
Plan plan_attend(int64_t requests, int64_t q_heads, int64_t kv_heads, int64_t head_dim, int64_t max_new, int64_t max_len) {
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
        const int64_t resident = resident_many(head_dim);
        // eight waves to a tile (each converts half as much) where that still leaves
        // two workgroups to a compute unit, one after the other: 4096 tokens of 32
        // heads 172 us against 188; 4 chunks of 300 tokens 167 against 161
        const bool wide = head_dim <= 128 && requests * kv_heads * ((rows + 255) / 256) >= resident;
        p.many.rows = wide ? 256 : 128;
        if (p.few.on) p.many.min_rows = kFewRows + 1;
        const int64_t sequences = requests * kv_heads * ((rows + 127) / 128);
        finish_part(&p.many, requests, kv_heads, head_dim, rows, max_len, resident,
                    wide || max_len <= (4 * sequences >= resident ? 2 : 1) * kWholeTokens || 2 * sequences >= resident);
    }
    return p;
}

// At least the bytes of plan_attend for every smaller number of requests, max_new
// and max_len too, which need not be less: a prompt of 4096 tokens of 32 heads is
// whole and needs none, 64 tokens behind as many share their work.  Work is
// shared out past kWholeTokens alone, by up to 64 rows of fewer than 8 * resident
// sequences and by 128-row tiles of fewer than resident / 2.
size_t workspace_bound(int64_t requests, int64_t q_heads, int64_t kv_heads, int64_t head_dim, int64_t max_new, int64_t max_len) {
    if (max_len <= kWholeTokens) return 0;
    const int64_t rows = max_new * (q_heads / kv_heads), units = (max_len + 255) / 256;
    auto part = [&](int64_t tile, int64_t most, int64_t limit, int64_t resident) {
        const int64_t sequences = std::min(requests * kv_heads * std::max<int64_t>(1, (most + tile - 1) / tile), limit);
        return part_bytes(std::min(resident, sequences * units), tile, sequences, head_dim);
    };
    size_t bytes = part(16, std::min<int64_t>(rows, 2 * kFewRows), 8 * resident_few(head_dim), resident_few(head_dim));
    if (rows > 2 * kFewRows) bytes += part(128, rows, resident_many(head_dim) / 2, resident_many(head_dim));
    return bytes;
}

// Launches one part of a call: W where a workgroup has a whole sequence, S where
// the work is shared out.
template <class W, class S>
int launch_part(AttendArgs a, const Part& p, int64_t blocks, int64_t max_rows, char* workspace, hipStream_t s) {
    if (!p.on) return GDSLLM_OK;
    a.min_rows = p.min_rows;
    a.max_rows = p.max_rows;
    a.tiles = p.tiles;
    a.part_o = reinterpret_cast<float*>(workspace);
    a.part_ml = reinterpret_cast<float2*>(a.part_o + p.sums * S::kD);
    a.parts = reinterpret_cast<int2*>(a.part_ml + p.sums);
    a.groups = p.sequences * blocks < (int64_t(1) << 30) ? p.groups : 0;  // the line of blocks is counted in 32 bits
    const unsigned per_request = static_cast<unsigned>(p.tiles) * a.c.kv_heads, requests = a.requests;
    if (a.groups == 0) {
        const size_t lds = sizeof(typename W::Lds);
        if (int rc = prepare_lds(reinterpret_cast<const void*>(&attend_whole<W>), lds)) return rc;
        hipLaunchKernelGGL(attend_whole<W>, dim3(per_request, requests), dim3(W::kThreads), lds, s, a);
        return check_hip(hipGetLastError(), "kv_attention launch");
    }
    const size_t lds = sizeof(typename S::Lds);
    if (int rc = prepare_lds(reinterpret_cast<const void*>(&attend_shared<S>), lds)) return rc;
    hipLaunchKernelGGL(attend_shared<S>, dim3(a.groups), dim3(256), lds, s, a);
    const int rows = static_cast<int>(std::min<int64_t>(S::kRows, std::max<int64_t>(1, max_rows)));
    const dim3 join(per_request * rows, requests);
    // few sequences are long, in many parts each
    if (p.sequences * rows <= kCus)
        hipLaunchKernelGGL((attend_join<S::kRows, S::kD, 1024>), join, dim3(1024), 0, s, a, rows);
    else
        hipLaunchKernelGGL((attend_join<S::kRows, S::kD, 256>), join, dim3(256), 0, s, a, rows);
    return check_hip(hipGetLastError(), "kv_attention launch");
}

template <bool E4M3, int D>
int launch_attend(AttendArgs a, const Plan& p, int64_t blocks, int64_t max_rows, char* workspace, hipStream_t s) {
    const int zero_other = a.zero_other;
    a.zero_other = p.few.on ? zero_other : 0;
    if (int rc = launch_part<RowTile<E4M3, D, 8>, RowTile<E4M3, D, 4>>(a, p.few, blocks, p.many.on ? kFewRows : max_rows, workspace, s))
        return rc;
    a.zero_other = p.few.on ? 0 : zero_other;
    char* ws = workspace + p.few.bytes;
    if constexpr (D <= 128)
        if (p.many.rows == 256) return launch_part<PromptTile<E4M3, D, 8>, PromptTile<E4M3, D, 4>>(a, p.many, blocks, max_rows, ws, s);
    return launch_part<PromptTile<E4M3, D, 4>, PromptTile<E4M3, D, 4>>(a, p.many, blocks, max_rows, ws, s);
}

bool attend_sizes(int64_t requests, int64_t q_heads, int64_t kv_heads, int64_t head_dim, int64_t max_new, int64_t max_len) {
    return requests >= 0 && requests <= 65535 && kv_heads >= 1 && kv_heads <= 1024 && q_heads >= kv_heads &&
           q_heads <= 16384 && q_heads % kv_heads == 0 && (head_dim == 64 || head_dim == 128 || head_dim == 256) &&
           max_new >= 0 && max_new <= (int64_t(1) << 24) && max_len >= 0 && max_len < (int64_t(1) << 31);
}

}  // namespace
}  // namespace gdsllm

using namespace gdsllm;

extern "C" size_t gdsllm_kv_attention_workspace_size(int64_t requests, int64_t q_heads, int64_t kv_heads,
                                                     int64_t head_dim, int64_t max_new, int64_t max_len) {
    if (!attend_sizes(requests, q_heads, kv_heads, head_dim, max_new, max_len)) return 0;
    return workspace_bound(requests, q_heads, kv_heads, head_dim, max_new, max_len);
}

extern "C" int gdsllm_kv_attention(const gdsllm_kv_cache8* cache, const void* q, int64_t ldq, void* o, int64_t ldo,
                                   int64_t tokens, int64_t q_heads, const int32_t* block_tables, int64_t table_width,
                                   int64_t ld_table, const int32_t* lens, const int32_t* starts, int64_t requests,
                                   float scale, int64_t max_new, int64_t max_len, int zero_other, void* workspace,
                                   size_t workspace_bytes, void* stream) {
    const std::string n = "kv_attention";
    auto bad = [&](const std::string& m) { return set_error(GDSLLM_ERR_INVALID_ARGUMENT, n + ": " + m); };
    AttendArgs a{};
    if (int rc = kv_cache_args(cache, n, &a.c)) return rc;
    const int64_t D = cache->head_dim;
    if (tokens < 0 || tokens > (int64_t(1) << 30)) return bad("bad token count");
    if (q_heads < 1 || q_heads % cache->kv_heads) return bad("q_heads must be a multiple of kv_heads");
    if (requests < 0 || requests > 65535) return bad("requests must be in [0, 65535]");
    if (table_width < 1 || ld_table < table_width) return bad("ld_table < table_width or an empty table");
    if (table_width > ((int64_t(1) << 31) - 1) / cache->block_size) return bad("table_width too large");
    if (max_new < 0 || max_len < 0) return bad("negative max_new or max_len");
    if (!(scale > 0.f) || scale > 1e30f) return bad("scale must be positive and finite");
    if (tokens == 0) return ok();
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
    const Plan p = plan_attend(requests, q_heads, cache->kv_heads, D, max_new, max_len);
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
    const int64_t max_rows = max_new * a.group;
    if (tokens * q_heads > (int64_t(1) << 30)) return bad("tokens * q_heads must be at most 2^30");
    const int64_t blocks = most / kBlock + 1;
    const bool e4m3 = cache->format == GDSLLM_KV_E4M3;
    const hipStream_t s = as_stream(stream);
    char* ws = static_cast<char*>(workspace);
    int rc = GDSLLM_OK;
#define GDSLLM_ATTEND(DIM)                                                          \
    if (D == DIM)                                                                   \
        rc = e4m3 ? launch_attend<true, DIM>(a, p, blocks, max_rows, ws, s)           \
                  : launch_attend<false, DIM>(a, p, blocks, max_rows, ws, s);
    GDSLLM_ATTEND(64)
    GDSLLM_ATTEND(128)
    GDSLLM_ATTEND(256)
#undef GDSLLM_ATTEND
    return rc ? rc : ok();
}
