// Attention over the 8-bit KV cache (kv_cache.hip writes it).
//
// For query row t of request b (n_b rows in this call, len_b tokens held) and
// query head h of kv head h / G:
//   x_j = scale * k_scale * (q . code_j),  j <= len_b - n_b + t
//   o   = sum_j 2^(x_j log2 e) v_j / sum_j 2^(x_j log2 e)
// in one pass over the tokens with a running maximum.  Codes enter the matrix
// cores as the fp16 values they are, so the products q . code and P . code are
// exact and summed in fp32; the scales stay outside: a block's key scale
// multiplies its scores, and its value scale is carried in the exponent.  With
// e = log2(v_scale) and the running maximum m taken over y_j = x_j log2 e + e,
//   acc += 2^(y_j - m) * code_j,   l += 2^(y_j - m) / v_scale,   o = acc / l,
// so the fp16 weights 2^(y_j - m) <= 1 lose nothing to a block whose values are
// large or small, whatever the other blocks' scales are.
//
// The G query heads of a kv head and the query rows share its keys: they are
// the 16 columns of one matrix tile (row r = token r / G, head r % G).

#include <algorithm>

#include "kv_cache.h"

namespace gdsllm {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kSegment = 4096;       // tokens whose block table a workgroup holds in LDS
constexpr int kMaxPages = kSegment / 16;
constexpr int kWaves = 4;

struct AttendArgs {
    KvCache c;
    const uint16_t* q;
    uint16_t* o;
    const int32_t *tables, *lens, *starts;
    float* part_o;   // [unit][16][D]
    float* part_ml;  // [unit][16][2]
    int64_t ldq, ldo, ld_table;
    float scale_log2;  // scale * log2 e
    int tokens, requests, q_heads, group, width;
    int chunk, splits, tiles;  // tokens of a unit; units along a sequence; row tiles of a request that have units
    int zero_tail;             // rows behind the last request are set to zero
};

// What this workgroup computes: a request's rows and the keys they may see.
struct Rows {
    int start, n, len, rows;
    __device__ __forceinline__ Rows(const AttendArgs& a, int b) {
        start = min(max(a.starts[b], 0), a.tokens);
        n = min(max(a.starts[b + 1] - start, 0), a.tokens - start);
        const int64_t most = static_cast<int64_t>(a.width) << a.c.block_log2;
        len = static_cast<int>(min(static_cast<int64_t>(max(a.lens[b], 0)), most));
        rows = n * a.group;
    }
    // Keys that the last of rows [r0, r0 + count) sees.
    __device__ __forceinline__ int keys(const AttendArgs& a, int r0, int count) const {
        const int last = (min(r0 + count, rows) - 1) / a.group;
        return max(len - n + last + 1, 0);
    }
};

__device__ __forceinline__ int chunks_of(const AttendArgs& a, int tile, int keys) {
    if (tile >= a.tiles) return 1;
    return min(max((keys + a.chunk - 1) / a.chunk, 1), a.splits);
}

// v from the other half of the wave (lanes l and l + 32), and from the other
// 16 lanes of each half, combined with f.
template <class F>
__device__ __forceinline__ float over_groups(float v, F f) {
    v = f(v, __shfl_xor(v, 16));
    return f(v, __shfl_xor(v, 32));
}

// Units (split, kv head and row tile, request): 16 rows over one chunk of
// tokens.  Matrix tiles are 16x16x32 and nothing passes through LDS but the
// block table:
//  * scores S^T = K Q^T: lane l gives key row l % 16 and 16 of each 64 channels
//    (one 16-byte load; Q's operand takes the same order), and receives, for query l % 16, tokens 4 * group .. + 3 of each 16;
//  * O^T = V^T P^T: its B operand is exactly those eight weights of two score
//    tiles, in place; V's operand needs eight tokens of one channel in a lane:
//    lanes load D/16 channels of the eight tokens and transpose 4x4 bytes with
//    v_perm.
template <bool E4M3, int D>
__global__ __launch_bounds__(kWaves * 64) void attend_rows(AttendArgs a) {
    constexpr int KS = D / 32;               // score steps of 32 channels
    constexpr int DB = D / 16;               // channels of V a lane holds
    constexpr int VW = DB / 4;               // the same in dwords
    constexpr int NT = D == 256 ? 2 : 4;     // score tiles of 16 tokens in an iteration
    constexpr int TT = 16 * NT;
    __shared__ int s_id[kMaxPages];
    __shared__ float s_c[kMaxPages], s_e[kMaxPages], s_inv[kMaxPages];
    __shared__ float s_o[2][16][D];
    __shared__ float s_m[kWaves][16], s_l[kWaves][16];

    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, col = lane & 15, g = lane >> 4;
    const int split = blockIdx.x, head = blockIdx.y % a.c.kv_heads, tile0 = blockIdx.y / a.c.kv_heads, b = blockIdx.z;
    const int bl = a.c.block_log2;
    if (a.zero_tail) {
        const int64_t id = (static_cast<int64_t>(b) * gridDim.y + blockIdx.y) * gridDim.x + split;
        const int64_t groups = static_cast<int64_t>(gridDim.x) * gridDim.y * gridDim.z;
        for (int64_t t = min(max(a.starts[a.requests], 0), a.tokens) + id; t < a.tokens; t += groups)
            for (int i = tid; i < a.q_heads * D / 8; i += kWaves * 64)
                *reinterpret_cast<uint4*>(a.o + t * a.ldo + 8 * i) = make_uint4(0, 0, 0, 0);
    }
    const Rows R(a, b);
    for (int tile = tile0; tile * 16 < R.rows; tile += gridDim.y / a.c.kv_heads) {
        const int keys = R.keys(a, tile * 16, 16);
        const int chunks = chunks_of(a, tile, keys);
        if (split >= chunks) continue;
        const int k0 = split * a.chunk, k1 = split == chunks - 1 ? keys : min(k0 + a.chunk, keys);
        const int r = tile * 16 + col;
        const bool valid = r < R.rows;
        const int t_row = R.start + (valid ? r / a.group : 0), h_row = head * a.group + (valid ? r % a.group : 0);
        const int last = valid ? R.len - R.n + r / a.group : -1;  // last key this row sees
        const int all_see = R.len - R.n + tile * 16 / a.group;    // every row sees keys up to here

        half8_t qf[KS];
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            uint4 w = make_uint4(0, 0, 0, 0);
            if (valid) w = *reinterpret_cast<const uint4*>(a.q + t_row * a.ldq + h_row * D + 64 * (s / 2) + 16 * g + 8 * (s & 1));
            qf[s] = __builtin_bit_cast(half8_t, w);
        }
        float4_t acc[DB];
#pragma unroll
        for (int j = 0; j < DB; ++j) acc[j] = float4_t{0.f, 0.f, 0.f, 0.f};
        float m = -INFINITY, l = 0.f;

        for (int seg = k0; seg < k1; seg += kSegment) {
            const int seg_end = min(seg + kSegment, k1);
            __syncthreads();
            const int pages = ((min(seg + kSegment, (k1 + TT - 1) & ~(TT - 1)) - seg) + (1 << bl) - 1) >> bl;
            bool lost = false;
            for (int p = tid; p < pages; p += kWaves * 64) {
                const int page = (seg >> bl) + p;
                const int id = page < a.width && (page << bl) < k1 ? a.tables[b * a.ld_table + page] : -1;
                const bool ok = id >= 0 && id < a.c.num_blocks;
                const int64_t sc = static_cast<int64_t>(ok ? id : 0) * a.c.kv_heads + head;
                const float vs = fmaxf(a.c.v_scale[sc], 0x1p-64f);
                s_id[p] = ok ? id : 0;
                s_c[p] = a.c.k_scale[sc] * a.scale_log2;
                s_e[p] = log2f(vs);
                s_inv[p] = ok ? 1.f / vs : 0.f;
                lost |= !ok && (page << bl) < k1;
            }
            const bool some_lost = __syncthreads_or(lost);
            for (int base = seg + wave * TT; base < seg_end; base += kWaves * TT) {
                uint32_t kw[NT][D / 16];
                uint32_t vw[NT][4][VW];
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    const int p = (base - seg + 16 * t) >> bl, off = (base + 16 * t) & ((1 << bl) - 1);
                    const int64_t row = ((static_cast<int64_t>(s_id[p]) * a.c.kv_heads + head) << bl) + off;
                    const uint32_t* kp = reinterpret_cast<const uint32_t*>(a.c.k + (row + col) * D + 16 * g);
#pragma unroll
                    for (int i = 0; i < D / 64; ++i) {
                        const u32x4_t w = __builtin_nontemporal_load(reinterpret_cast<const u32x4_t*>(kp + 16 * i));
#pragma unroll
                        for (int j = 0; j < 4; ++j) kw[t][4 * i + j] = w[j];
                    }
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const uint8_t* vp = a.c.v + (row + 4 * g + i) * D + col * DB;
                        if constexpr (VW == 1) {
                            vw[t][i][0] = __builtin_nontemporal_load(reinterpret_cast<const uint32_t*>(vp));
                        } else if constexpr (VW == 2) {
                            const uint64_t w = __builtin_nontemporal_load(reinterpret_cast<const uint64_t*>(vp));
                            vw[t][i][0] = static_cast<uint32_t>(w);
                            vw[t][i][1] = static_cast<uint32_t>(w >> 32);
                        } else {
                            const u32x4_t w = __builtin_nontemporal_load(reinterpret_cast<const u32x4_t*>(vp));
#pragma unroll
                            for (int j = 0; j < 4; ++j) vw[t][i][j] = w[j];
                        }
                    }
                }
                float x[NT][4];
                float mx = -INFINITY;
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    float4_t s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int i = 0; i < KS; ++i) {
                        uint32_t f[4];
                        codes_to_f16<E4M3>(kw[t][2 * i], f[0], f[1]);
                        codes_to_f16<E4M3>(kw[t][2 * i + 1], f[2], f[3]);
                        const half8_t kf = __builtin_bit_cast(half8_t, make_uint4(f[0], f[1], f[2], f[3]));
                        s = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, qf[i], s, 0, 0, 0);
                    }
                    const int p = (base - seg + 16 * t) >> bl;
                    const float c = s_c[p], e = s_e[p];
#pragma unroll
                    for (int i = 0; i < 4; ++i) x[t][i] = fmaf(s[i], c, e);
                }
                if (base + TT - 1 > all_see || base + TT > k1 || some_lost) {
#pragma unroll
                    for (int t = 0; t < NT; ++t) {
                        // a block outside the cache has no weight
                        const bool none = s_inv[(base - seg + 16 * t) >> bl] == 0.f;
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const int j = base + 16 * t + 4 * g + i;
                            if (j > last || j >= k1 || none) x[t][i] = -INFINITY;
                            if (j >= k1 || none) {  // what lies there may be no number
#pragma unroll
                                for (int w = 0; w < VW; ++w) vw[t][i][w] = 0;
                            }
                        }
                    }
                }
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int i = 0; i < 4; ++i) mx = fmaxf(mx, x[t][i]);
                mx = over_groups(mx, [](float u, float v) { return fmaxf(u, v); });
                const float m_new = fmaxf(m, mx);
                const float ref = m_new == -INFINITY ? 0.f : m_new;
                if (__any(m_new > m)) {
                    const float alpha = __builtin_amdgcn_exp2f(m - ref);
                    l *= alpha;
#pragma unroll
                    for (int j = 0; j < DB; ++j) acc[j] *= alpha;
                    m = m_new;
                }
                half8_t pf[NT / 2];
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    const float inv = s_inv[(base - seg + 16 * t) >> bl];
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
                    for (int w = 0; w < VW; ++w) {
                        // pairs[k]: tokens 2k, 2k+1 of the eight, channels 0, 1 (lo) and 2, 3 (hi)
                        uint32_t f[4][4];  // [channel][token pair]
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            const uint32_t t0 = vw[2 * u + k / 2][2 * (k & 1)][w], t1 = vw[2 * u + k / 2][2 * (k & 1) + 1][w];
                            codes_to_f16<E4M3>(__builtin_amdgcn_perm(t1, t0, 0x05010400u), f[0][k], f[1][k]);
                            codes_to_f16<E4M3>(__builtin_amdgcn_perm(t1, t0, 0x07030602u), f[2][k], f[3][k]);
                        }
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const half8_t vf = __builtin_bit_cast(half8_t, make_uint4(f[j][0], f[j][1], f[j][2], f[j][3]));
                            acc[4 * w + j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, pf[u], acc[4 * w + j], 0, 0, 0);
                        }
                    }
            }
        }
        l = over_groups(l, [](float u, float v) { return u + v; });

        // the four waves' sums, in a fixed order: (0 + 2) + (1 + 3)
        if (g == 0) {
            s_m[wave][col] = m;
            s_l[wave][col] = l;
        }
        __syncthreads();
        float mw = s_m[0][col];
#pragma unroll
        for (int w = 1; w < kWaves; ++w) mw = fmaxf(mw, s_m[w][col]);
        const float ref = mw == -INFINITY ? 0.f : mw;
        const float f = __builtin_amdgcn_exp2f(m - ref);
        l = 0.f;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) l = fmaf(s_l[w][col], __builtin_amdgcn_exp2f(s_m[w][col] - ref), l);
#pragma unroll
        for (int j = 0; j < DB; ++j) acc[j] *= f;
        auto put = [&](float (*o)[D]) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < DB; j += 4)
                    *reinterpret_cast<float4_t*>(&o[col][(4 * g + i) * DB + j]) =
                        float4_t{acc[j][i], acc[j + 1][i], acc[j + 2][i], acc[j + 3][i]};
        };
        auto add = [&](float (*o)[D]) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < DB; ++j) acc[j][i] += o[col][(4 * g + i) * DB + j];
        };
        if (wave >= 2) put(s_o[wave - 2]);
        __syncthreads();
        if (wave < 2) add(s_o[wave]);
        __syncthreads();
        if (wave == 1) put(s_o[0]);
        __syncthreads();
        if (wave == 0) {
            add(s_o[0]);
            if (chunks == 1) {
                if (valid) {
                    const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
                    uint16_t* o = a.o + t_row * a.ldo + h_row * D;
#pragma unroll
                    for (int i = 0; i < 4; ++i)
#pragma unroll
                        for (int j = 0; j < DB; j += 4) {
                            uint2 w;
                            w.x = pack_h2(static_cast<half_t>(acc[j][i] * inv), static_cast<half_t>(acc[j + 1][i] * inv));
                            w.y = pack_h2(static_cast<half_t>(acc[j + 2][i] * inv), static_cast<half_t>(acc[j + 3][i] * inv));
                            *reinterpret_cast<uint2*>(o + (4 * g + i) * DB + j) = w;
                        }
                }
            } else if (valid) {
                const int64_t unit = ((static_cast<int64_t>(b) * a.tiles + tile) * a.c.kv_heads + head) * a.splits + split;
                float* o = a.part_o + (unit * 16 + col) * D;
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int j = 0; j < DB; j += 4)
                        *reinterpret_cast<float4_t*>(o + (4 * g + i) * DB + j) =
                            float4_t{acc[j][i], acc[j + 1][i], acc[j + 2][i], acc[j + 3][i]};
                if (g == 0) {
                    a.part_ml[(unit * 16 + col) * 2] = mw;
                    a.part_ml[(unit * 16 + col) * 2 + 1] = l;
                }
            }
        }
    }
}

// Rows whose tokens were split: their units' sums joined in order.
template <int D>
__global__ __launch_bounds__(256) void attend_join(AttendArgs a) {
    constexpr int TPR = D / 4;  // threads of a row
    const int head = blockIdx.x % a.c.kv_heads, tile = blockIdx.x / a.c.kv_heads, b = blockIdx.y;
    const Rows R(a, b);
    if (tile * 16 >= R.rows) return;
    const int chunks = chunks_of(a, tile, R.keys(a, tile * 16, 16));
    if (chunks == 1) return;
    const int64_t unit = ((static_cast<int64_t>(b) * a.tiles + tile) * a.c.kv_heads + head) * a.splits;
    const int d = 4 * (threadIdx.x % TPR);
    for (int r = threadIdx.x / TPR; r < 16 && tile * 16 + r < R.rows; r += 256 / TPR) {
        const float* ml = a.part_ml + (unit * 16 + r) * 2;
        float m = -INFINITY;
        for (int s = 0; s < chunks; ++s) m = fmaxf(m, ml[s * 32]);
        const float ref = m == -INFINITY ? 0.f : m;
        float l = 0.f;
        float4_t o = {0.f, 0.f, 0.f, 0.f};
        for (int s = 0; s < chunks; ++s) {
            const float f = __builtin_amdgcn_exp2f(ml[s * 32] - ref);
            l = fmaf(ml[s * 32 + 1], f, l);
            const float4_t p = *reinterpret_cast<const float4_t*>(a.part_o + ((unit + s) * 16 + r) * D + d);
            o += p * f;
        }
        const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
        const int row = tile * 16 + r;
        uint16_t* out = a.o + (R.start + row / a.group) * a.ldo + (head * a.group + row % a.group) * D + d;
        uint2 w;
        w.x = pack_h2(static_cast<half_t>(o[0] * inv), static_cast<half_t>(o[1] * inv));
        w.y = pack_h2(static_cast<half_t>(o[2] * inv), static_cast<half_t>(o[3] * inv));
        *reinterpret_cast<uint2*>(out) = w;
    }
}

struct Plan {
    int tiles, splits, chunk;
    int64_t units;
};

// Row tiles, chunk length and units of a call.  Enough units to give every
// compute unit a few workgroups, none shorter than 256 tokens.
Plan plan_attend(int64_t requests, int64_t q_heads, int64_t kv_heads, int64_t max_new, int64_t max_len) {
    Plan p;
    p.tiles = static_cast<int>(std::max<int64_t>(1, (max_new * (q_heads / kv_heads) + 15) / 16));
    const int64_t lanes = requests * kv_heads * p.tiles;
    int64_t chunk = (max_len * lanes / 1024 + 255) / 256 * 256;
    chunk = std::min<int64_t>(std::max<int64_t>(chunk, 256), kSegment);
    p.chunk = static_cast<int>(chunk);
    p.splits = static_cast<int>(std::max<int64_t>(1, (max_len + chunk - 1) / chunk));
    p.units = p.splits > 1 ? lanes * p.splits : 0;
    return p;
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
    return static_cast<size_t>(plan_attend(requests, q_heads, kv_heads, max_new, max_len).units) * 16 *
           (head_dim + 2) * sizeof(float);
}

extern "C" int gdsllm_kv_attention(const gdsllm_kv_cache8* cache, const void* q, int64_t ldq, void* o, int64_t ldo,
                                   int64_t tokens, int64_t q_heads, const int32_t* block_tables, int64_t table_width,
                                   int64_t ld_table, const int32_t* lens, const int32_t* starts, int64_t requests,
                                   float scale, int64_t max_new, int64_t max_len, int zero_tail, void* workspace,
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
    const Plan p = plan_attend(requests, q_heads, cache->kv_heads, max_new, max_len);
    const size_t need = static_cast<size_t>(p.units) * 16 * (D + 2) * sizeof(float);
    if (need > 0 && (!workspace || workspace_bytes < need))
        return bad("workspace of " + std::to_string(need) + " bytes needed, got " + std::to_string(workspace_bytes));
    a.q = static_cast<const uint16_t*>(q);
    a.o = static_cast<uint16_t*>(o);
    a.tables = block_tables;
    a.lens = lens;
    a.starts = starts;
    a.part_o = static_cast<float*>(workspace);
    a.part_ml = a.part_o + p.units * 16 * D;
    a.ldq = ldq;
    a.ldo = ldo;
    a.ld_table = ld_table;
    a.scale_log2 = scale * kLog2e;
    a.tokens = static_cast<int>(tokens);
    a.requests = static_cast<int>(requests);
    a.q_heads = static_cast<int>(q_heads);
    a.group = static_cast<int>(q_heads / cache->kv_heads);
    a.width = static_cast<int>(table_width);
    a.chunk = p.chunk;
    a.splits = p.splits;
    a.tiles = p.tiles;
    a.zero_tail = zero_tail;
    const int64_t y = std::min<int64_t>(p.tiles, 65535 / cache->kv_heads) * cache->kv_heads;
    const dim3 grid(static_cast<unsigned>(p.splits), static_cast<unsigned>(y), static_cast<unsigned>(requests));
    const bool e4m3 = cache->format == GDSLLM_KV_E4M3;
    const hipStream_t s = as_stream(stream);
#define GDSLLM_ATTEND(DIM)                                                                            \
    if (D == DIM) {                                                                                   \
        if (e4m3) hipLaunchKernelGGL((attend_rows<true, DIM>), grid, dim3(kWaves * 64), 0, s, a);     \
        else hipLaunchKernelGGL((attend_rows<false, DIM>), grid, dim3(kWaves * 64), 0, s, a);         \
        if (p.splits > 1)                                                                             \
            hipLaunchKernelGGL(attend_join<DIM>, dim3(static_cast<unsigned>(p.tiles * cache->kv_heads), \
                                                      static_cast<unsigned>(requests)), dim3(256), 0, s, a); \
    }
    GDSLLM_ATTEND(64)
    GDSLLM_ATTEND(128)
    GDSLLM_ATTEND(256)
#undef GDSLLM_ATTEND
    if (int rc = check_hip(hipGetLastError(), "kv_attention launch")) return rc;
    return ok();
}
