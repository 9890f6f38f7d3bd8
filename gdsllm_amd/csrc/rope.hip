// Rotary positions: q and k turned by their tokens' positions (gdsllm_rope).
//
// For pair i of a head, channels (a, b) = (i, i + R/2) of the first R (halves) or
// (2i, 2i + 1) (neighbours), and angle phi = angle[position][i]:
//   y_a = x_a cos phi - x_b sin phi,   y_b = x_b cos phi + x_a sin phi,
// in 64 bits, rounded to fp32 and fp16.  The other channels are copied.  Bound by
// the bytes of q and k, read and written once: 4001 tokens of 64 heads of 128
// channels 26.5 us, 5.0 TB/s, from memory (stores that stay in the caches: 29.2).

#include <algorithm>

#include "rope.h"

namespace gdsllm {
namespace {

struct RopeArgs {
    RopeRows r;
    const int32_t* positions;
    const float *cos, *sin;
    int64_t tokens;
    int D, half, max_pos;
    int units, share;  // units of a head; threads groups of `units` that share a token's heads
};

// Groups of `units` threads, `share` of them to a token; each takes HEADS heads.
template <bool NEIGHBOURS, int HEADS>
__global__ __launch_bounds__(256) void rope_chunks(RopeArgs a) {
    const int per = 256 / a.units, g = threadIdx.x / a.units;
    if (g >= per) return;
    const int64_t group = static_cast<int64_t>(blockIdx.x) * per + g, t = group / a.share;
    if (t >= a.tokens) return;
    const int pos = a.positions[t];
    const bool live = static_cast<uint32_t>(pos) < static_cast<uint32_t>(a.max_pos);
    const int64_t at = live ? static_cast<int64_t>(pos) * a.half : 0;
    rope_unit<NEIGHBOURS, HEADS>(a.r, a.D, a.half, t, threadIdx.x - g * a.units, static_cast<int>(group - t * a.share), a.share,
                                 live, a.cos + at, a.sin + at);
}

// Any even rotary part, any head_dim, rows and pointers off the 16-byte grid: a
// pair, or a channel that stays, to a thread.
template <bool NEIGHBOURS>
__global__ __launch_bounds__(256) void rope_pairs(RopeArgs a) {
    const int64_t per_head = a.D - a.half, n = a.tokens * a.r.heads * per_head;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < n; i += static_cast<int64_t>(gridDim.x) * 256) {
        const int64_t row = i / per_head, t = row / a.r.heads;
        const int p = static_cast<int>(i - row * per_head), h = static_cast<int>(row - t * a.r.heads);
        const int pos = a.positions[t];
        const bool live = static_cast<uint32_t>(pos) < static_cast<uint32_t>(a.max_pos);
        const uint16_t* x = a.r.from(t, h, a.D);
        uint16_t* y = a.r.to(t, h, a.D);
        if (p >= a.half) {
            y[a.half + p] = live ? x[a.half + p] : 0;
            continue;
        }
        const int c0 = NEIGHBOURS ? 2 * p : p, c1 = NEIGHBOURS ? 2 * p + 1 : p + a.half;
        uint16_t r0 = 0, r1 = 0;
        if (live) {
            const int64_t at = static_cast<int64_t>(pos) * a.half + p;
            const double u = h2f(x[c0]), v = h2f(x[c1]), c = a.cos[at], s = a.sin[at];
            r0 = turned(u, c, -(v * s));
            r1 = turned(v, c, u * s);
        }
        y[c0] = r0;
        y[c1] = r1;
    }
}

// `tokens` rows of `width` halves, ld apart.
struct Span {
    const void* p;
    int64_t ld, width;
};

// Whether two of them share a byte.  Rows of one distance may lie between each
// other's (q and k in the rows of one projection); of different ones they are
// taken to meet where the memory from the first row to the last does.
bool meet(const Span& a, const Span& b, int64_t tokens) {
    const uint64_t pa = reinterpret_cast<uintptr_t>(a.p), pb = reinterpret_cast<uintptr_t>(b.p);
    auto bytes = [&](const Span& s) { return 2 * (static_cast<uint64_t>(tokens - 1) * s.ld + s.width); };
    if (pa >= pb + bytes(b) || pb >= pa + bytes(a)) return false;
    if (tokens == 1 || a.ld != b.ld) return true;
    const uint64_t period = 2 * static_cast<uint64_t>(a.ld);
    const uint64_t d = pb >= pa ? (pb - pa) % period : (period - (pa - pb) % period) % period;  // of b's row from one of a
    return d < 2 * static_cast<uint64_t>(a.width) || d + 2 * static_cast<uint64_t>(b.width) > period;
}

}  // namespace
}  // namespace gdsllm

using namespace gdsllm;

extern "C" int gdsllm_rope(const void* q, int64_t ldq, void* q_out, int64_t ldqo, int64_t q_heads, const void* k, int64_t ldk,
                           void* k_out, int64_t ldko, int64_t k_heads, int64_t head_dim, int64_t tokens,
                           const int32_t* positions, const float* cos, const float* sin, int64_t rotary, int64_t max_pos,
                           int neighbours, void* stream) {
    const std::string n = "rope";
    auto bad = [&](const std::string& m) { return set_error(GDSLLM_ERR_INVALID_ARGUMENT, n + ": " + m); };
    if (head_dim < 2 || head_dim > 1024) return bad("head_dim must be in [2, 1024], got " + std::to_string(head_dim));
    if (rotary < 2 || rotary > head_dim || rotary % 2)
        return bad("rotary must be even and in [2, head_dim], got " + std::to_string(rotary));
    if (tokens < 0 || tokens > (int64_t(1) << 30)) return bad("bad token count");
    if (q_heads < 1 || q_heads > 16384) return bad("q_heads must be in [1, 16384]");
    if (k_heads < 0 || k_heads > 16384) return bad("k_heads must be in [0, 16384]");
    if (tokens == 0) return ok();
    if (!q || !q_out || (k_heads > 0 && (!k || !k_out)) || !positions || !cos || !sin) return bad("null pointer");
    if (max_pos < 1 || max_pos > (int64_t(1) << 31) - 1) return bad("bad number of positions");
    const bool has_k = k_heads > 0;
    if (tokens > 1 && (ldq < q_heads * head_dim || ldqo < q_heads * head_dim ||
                       (has_k && (ldk < k_heads * head_dim || ldko < k_heads * head_dim))))
        return bad("row stride smaller than a row");
    const uintptr_t rows = reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(q_out) |
                           (has_k ? reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(k_out) : 0);
    if (rows % 2 || (reinterpret_cast<uintptr_t>(positions) | reinterpret_cast<uintptr_t>(cos) |
                     reinterpret_cast<uintptr_t>(sin)) % 4)
        return bad("misaligned pointer");
    if ((q == q_out && tokens > 1 && ldq != ldqo) || (has_k && k == k_out && tokens > 1 && ldk != ldko))
        return bad("in place the strides must be equal");
    const Span qs{q, ldq, q_heads * head_dim}, qos{q_out, ldqo, qs.width}, ks{k, ldk, k_heads * head_dim}, kos{k_out, ldko, ks.width};
    if ((q != q_out && meet(qos, qs, tokens)) ||
        (has_k && ((k != k_out && meet(kos, ks, tokens)) || meet(qos, ks, tokens) || meet(kos, qs, tokens) || meet(qos, kos, tokens))))
        return bad("q_out and k_out must overlap neither each other nor q and k, but for q_out = q and k_out = k");
    RopeArgs a{};
    a.r = {static_cast<const uint16_t*>(q), static_cast<const uint16_t*>(k), static_cast<uint16_t*>(q_out),
           static_cast<uint16_t*>(k_out), ldq, ldk, ldqo, ldko, static_cast<int>(q_heads), static_cast<int>(q_heads + k_heads)};
    a.positions = positions;
    a.cos = cos;
    a.sin = sin;
    a.tokens = tokens;
    a.D = static_cast<int>(head_dim);
    a.half = static_cast<int>(rotary / 2);
    a.max_pos = static_cast<int>(max_pos);
    const hipStream_t s = as_stream(stream);
    const int64_t strides = tokens > 1 ? ldq | ldqo | (has_k ? ldk | ldko : 0) : 0;
    const uintptr_t tables = reinterpret_cast<uintptr_t>(cos) | reinterpret_cast<uintptr_t>(sin);
    const bool chunks = head_dim % 8 == 0 && rotary % (neighbours ? 8 : 16) == 0 && strides % 8 == 0 && rows % 16 == 0 &&
                        tables % 16 == 0;
    if (!chunks) {
        const int64_t items = tokens * a.r.heads * (head_dim - a.half);
        const int64_t grid = std::min<int64_t>((items + 255) / 256, 64 * static_cast<int64_t>(cu_count()));
        if (neighbours) hipLaunchKernelGGL(rope_pairs<true>, dim3(static_cast<unsigned>(grid)), dim3(256), 0, s, a);
        else hipLaunchKernelGGL(rope_pairs<false>, dim3(static_cast<unsigned>(grid)), dim3(256), 0, s, a);
        if (int rc = check_hip(hipGetLastError(), "rope launch")) return rc;
        return ok();
    }
    a.units = rope_units(a.D, a.half, neighbours != 0);
    const int per = 256 / a.units;
    // four heads to a thread where that leaves every compute unit work
    const int heads = tokens * a.r.heads >= 64 * static_cast<int64_t>(cu_count()) ? 4 : 1;
    a.share = (a.r.heads + heads - 1) / heads;
    const int64_t grid = (tokens * a.share + per - 1) / per;
    if (grid * 256 >= (int64_t(1) << 32)) return bad("too many tokens and heads for one call");
    const dim3 g(static_cast<unsigned>(grid));
    if (heads == 4) {
        if (neighbours) hipLaunchKernelGGL((rope_chunks<true, 4>), g, dim3(256), 0, s, a);
        else hipLaunchKernelGGL((rope_chunks<false, 4>), g, dim3(256), 0, s, a);
    } else {
        if (neighbours) hipLaunchKernelGGL((rope_chunks<true, 1>), g, dim3(256), 0, s, a);
        else hipLaunchKernelGGL((rope_chunks<false, 1>), g, dim3(256), 0, s, a);
    }
    if (int rc = check_hip(hipGetLastError(), "rope launch")) return rc;
    return ok();
}
