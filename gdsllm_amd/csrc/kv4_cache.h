// What the kernels over the 4-bit KV cache share: its layout and its codes.
#pragma once

#include "common.h"

namespace gdsllm {

// One layer's cache as the kernels take it (gdsllm_kv_cache4 with narrow sizes).
struct Kv4Cache {
    uint8_t* k;
    uint8_t* v;
    uint32_t* k_affine;  // (scale, bias) of [block][kv_head][group][token]
    uint32_t* v_affine;
    int num_blocks, kv_heads;
    int block_log2;      // log2(block_size)
    int group_log2;      // log2(channels of a group)
    int groups;          // groups of a head
};

// Checks `c` and narrows it; `where` names the caller in the message.
int kv4_cache_args(const gdsllm_kv_cache4* c, const std::string& where, Kv4Cache* out);

// Two codes as an exact fp16 pair, from words whose fields at bits [0,4) and
// [16,20) (low) or [4,8) and [20,24) (high) hold them: below the exponent of 1024
// (64) a code is 1024 + code (64 + code).
__device__ __forceinline__ half2_t codes_low(const NibUnpack& n, uint32_t w) {
    const half2_t off = {static_cast<half_t>(-1024.f), static_cast<half_t>(-1024.f)};
    return __builtin_bit_cast(half2_t, n.lo_c(w)) + off;
}
__device__ __forceinline__ half2_t codes_high(const NibUnpack& n, uint32_t w) {
    const half2_t off = {static_cast<half_t>(-64.f), static_cast<half_t>(-64.f)};
    return __builtin_bit_cast(half2_t, n.hi_c(w)) + off;
}
// code * scale + bias, rounded once.
__device__ __forceinline__ half2_t element2(half2_t code, half2_t scale, half2_t bias) {
    return __builtin_elementwise_fma(code, scale, bias);
}
__device__ __forceinline__ half2_t both(uint32_t w, bool high) {
    const half2_t x = __builtin_bit_cast(half2_t, w);
    return high ? half2_t{x.y, x.y} : half2_t{x.x, x.x};
}

// The eight elements of one dword of codes (channels 0 .. 7) of one group, as
// pairs (0, 4), (1, 5), (2, 6), (3, 7).
__device__ __forceinline__ uint4 elements8(const NibUnpack& n, uint32_t w, uint32_t affine) {
    const half2_t s = both(affine, false), b = both(affine, true);
    const uint32_t w8 = w >> 8;
    return make_uint4(__builtin_bit_cast(uint32_t, element2(codes_low(n, w), s, b)),
                      __builtin_bit_cast(uint32_t, element2(codes_high(n, w), s, b)),
                      __builtin_bit_cast(uint32_t, element2(codes_low(n, w8), s, b)),
                      __builtin_bit_cast(uint32_t, element2(codes_high(n, w8), s, b)));
}
// Eight fp16 values 0 .. 7 from that order to rising order, and back.
__device__ __forceinline__ uint4 rising_from_pairs(const uint4& p) {
    return make_uint4(__builtin_amdgcn_perm(p.y, p.x, 0x05040100u), __builtin_amdgcn_perm(p.w, p.z, 0x05040100u),
                      __builtin_amdgcn_perm(p.y, p.x, 0x07060302u), __builtin_amdgcn_perm(p.w, p.z, 0x07060302u));
}
__device__ __forceinline__ uint4 pairs_from_rising(const uint4& x) {
    return make_uint4(__builtin_amdgcn_perm(x.z, x.x, 0x05040100u), __builtin_amdgcn_perm(x.z, x.x, 0x07060302u),
                      __builtin_amdgcn_perm(x.w, x.y, 0x05040100u), __builtin_amdgcn_perm(x.w, x.y, 0x07060302u));
}

}  // namespace gdsllm
