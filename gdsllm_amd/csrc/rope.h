// Rotation of channel pairs by an angle, for the kernels that turn q and k.
#pragma once

#include "common.h"

namespace gdsllm {

// One rotated value own * c + other * s (s negated by the caller for the first
// of a pair): in 64 bits, where the products of an fp16 and an fp32 value are
// exact; then to fp32 and from there to fp16, as torch's own cast from 64 bits
// goes (a value within 2^-25 of itself of the middle between two fp16 values may
// go to the farther one).
__device__ __forceinline__ uint16_t turned(double own, double c, double other_s) {
    return f2h_bits(fp32_rounded(static_cast<float>(fma(own, c, other_s))));
}

// Eight channels as halves of a 16-byte chunk.
__device__ __forceinline__ uint16_t half_of(const uint4& x, int j) {
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
    return static_cast<uint16_t>(w[j / 2] >> (16 * (j & 1)));
}
__device__ __forceinline__ uint4 pack8(const uint16_t (&h)[8]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = h[2 * i] | (static_cast<uint32_t>(h[2 * i + 1]) << 16);
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// Cosines and sines of N angles, 16-byte aligned.
template <int N>
struct Angles {
    float4_t c[N / 4], s[N / 4];
    __device__ __forceinline__ void load(const float* cos, const float* sin) {
#pragma unroll
        for (int i = 0; i < N / 4; ++i) {
            c[i] = *reinterpret_cast<const float4_t*>(cos + 4 * i);
            s[i] = *reinterpret_cast<const float4_t*>(sin + 4 * i);
        }
    }
    __device__ __forceinline__ double cos_of(int i) const { return c[i / 4][i % 4]; }
    __device__ __forceinline__ double sin_of(int i) const { return s[i / 4][i % 4]; }
};

// Halves: pair i is channel i of `lo` and of `hi`.
__device__ __forceinline__ void turn_halves(uint4& lo, uint4& hi, const Angles<8>& t) {
    uint16_t a[8], b[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const double x = h2f(half_of(lo, j)), y = h2f(half_of(hi, j)), c = t.cos_of(j), s = t.sin_of(j);
        a[j] = turned(x, c, -(y * s));
        b[j] = turned(y, c, x * s);
    }
    lo = pack8(a);
    hi = pack8(b);
}
// One half of that: the rotated `own`, which is the first half's chunk or the second's.
__device__ __forceinline__ uint4 turn_half(const uint4& own, const uint4& other, bool first, const Angles<8>& t) {
    uint16_t r[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const double os = static_cast<double>(h2f(half_of(other, j))) * t.sin_of(j);
        r[j] = turned(h2f(half_of(own, j)), t.cos_of(j), first ? -os : os);
    }
    return pack8(r);
}
// Neighbours: pair i is channels 2i and 2i + 1.
__device__ __forceinline__ uint4 turn_neighbours(const uint4& x, const Angles<4>& t) {
    uint16_t r[8];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const double a = h2f(half_of(x, 2 * j)), b = h2f(half_of(x, 2 * j + 1)), c = t.cos_of(j), s = t.sin_of(j);
        r[2 * j] = turned(a, c, -(b * s));
        r[2 * j + 1] = turned(b, c, a * s);
    }
    return pack8(r);
}

// Heads of one or two tensors (q, then k) to rotate into others, rows ldx apart.
struct RopeRows {
    const uint16_t *q, *k;
    uint16_t *q_out, *k_out;
    int64_t ldq, ldk, ldqo, ldko;
    int q_heads, heads;  // heads: of both
    __device__ __forceinline__ const uint16_t* from(int64_t t, int h, int D) const {
        return h < q_heads ? q + t * ldq + static_cast<int64_t>(h) * D : k + t * ldk + static_cast<int64_t>(h - q_heads) * D;
    }
    __device__ __forceinline__ uint16_t* to(int64_t t, int h, int D) const {
        return h < q_heads ? q_out + t * ldqo + static_cast<int64_t>(h) * D : k_out + t * ldko + static_cast<int64_t>(h - q_heads) * D;
    }
};

// Unit u of heads h0, h0 + step, ... (HEADS of them at most) of token t, by one
// thread.  A head has `turns` units that rotate (eight pairs of halves, four of
// neighbours) and then one for each chunk of eight channels that stays; all
// loads are issued before the first rotation.  A row without a position is zero.
template <bool NEIGHBOURS, int HEADS>
__device__ __forceinline__ void rope_unit(const RopeRows& r, int D, int half, int64_t t, int u, int h0, int step, bool live,
                                          const float* cos, const float* sin) {
    const int turns = NEIGHBOURS ? half >> 2 : half >> 3;
    const bool rotates = u < turns;
    // first channel of the unit's chunk, and of its second one
    const int c0 = rotates || NEIGHBOURS ? 8 * u : 2 * half + 8 * (u - turns), c1 = c0 + half;
    uint4 x[HEADS], y[HEADS];
#pragma unroll
    for (int i = 0; i < HEADS; ++i) {
        const int h = h0 + i * step;
        x[i] = y[i] = make_uint4(0, 0, 0, 0);
        if (live && h < r.heads) {
            const uint16_t* p = r.from(t, h, D);
            x[i] = *reinterpret_cast<const uint4*>(p + c0);
            if (!NEIGHBOURS && rotates) y[i] = *reinterpret_cast<const uint4*>(p + c1);
        }
    }
    if (live && rotates) {
        Angles<NEIGHBOURS ? 4 : 8> a;
        a.load(cos + (NEIGHBOURS ? 4 : 8) * u, sin + (NEIGHBOURS ? 4 : 8) * u);
#pragma unroll
        for (int i = 0; i < HEADS; ++i) {
            if constexpr (NEIGHBOURS) x[i] = turn_neighbours(x[i], a);
            else turn_halves(x[i], y[i], a);
        }
    }
#pragma unroll
    for (int i = 0; i < HEADS; ++i) {
        const int h = h0 + i * step;
        if (h >= r.heads) continue;
        uint16_t* p = r.to(t, h, D);
        store_nt16(p + c0, x[i]);
        if (!NEIGHBOURS && rotates) store_nt16(p + c1, y[i]);
    }
}

// Units of a head of D channels, `half` of them in one half of the rotated part.
__host__ __device__ inline int rope_units(int D, int half, bool neighbours) { return D / 8 - (neighbours ? 0 : half / 8); }

}  // namespace gdsllm
