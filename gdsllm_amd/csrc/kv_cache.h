// What the kernels over the 8-bit KV cache share: its layout and its codes.
#pragma once

#include "common.h"

namespace gdsllm {

// One layer's cache as the kernels take it (gdsllm_kv_cache8 with narrow sizes).
struct KvCache {
    uint8_t* k;
    uint8_t* v;
    float* k_scale;
    float* v_scale;
    int num_blocks, kv_heads;
    int block_log2;  // log2(block_size)
};

// Checks `c` and narrows it; `where` names the caller in the message.
int kv_cache_args(const gdsllm_kv_cache8* c, const std::string& where, KvCache* out);

constexpr float kE4m3Max = 448.f;  // largest finite e4m3 code
constexpr float kInt8Max = 127.f;

// Four codes (one dword) as two packed fp16 pairs, exactly: both e4m3 and int8
// values are fp16 values.
template <bool E4M3>
__device__ __forceinline__ void codes_to_f16(uint32_t w, uint32_t& lo, uint32_t& hi) {
    if constexpr (E4M3) {
        lo = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, false));
        hi = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, true));
    } else {
        // byte ^ 0x80 is code + 128; below the exponent byte 0x64 it is the fp16
        // value 1024 + 128 + code
        const uint32_t u = w ^ 0x80808080u;
        const half2_t off = {static_cast<half_t>(1152.f), static_cast<half_t>(1152.f)};
        const uint32_t a = __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u);
        const uint32_t b = __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u);
        lo = __builtin_bit_cast(uint32_t, __builtin_bit_cast(half2_t, a) - off);
        hi = __builtin_bit_cast(uint32_t, __builtin_bit_cast(half2_t, b) - off);
    }
}

// The code nearest to x (ties to even), saturated; NaN stays NaN in e4m3 and
// becomes 0 in int8.  Four values to one dword.
template <bool E4M3>
__device__ __forceinline__ uint32_t to_codes(float a, float b, float c, float d) {
    if constexpr (E4M3) {
        auto sat = [](float x) { return x == x ? fminf(fmaxf(x, -kE4m3Max), kE4m3Max) : x; };
        int r = __builtin_amdgcn_cvt_pk_fp8_f32(sat(a), sat(b), 0, false);
        r = __builtin_amdgcn_cvt_pk_fp8_f32(sat(c), sat(d), r, true);
        return static_cast<uint32_t>(r);
    } else {
        auto q = [](float x) {
            const float r = x == x ? fminf(fmaxf(__builtin_rintf(x), -kInt8Max), kInt8Max) : 0.f;
            return static_cast<uint32_t>(static_cast<int>(r)) & 0xFFu;
        };
        return q(a) | (q(b) << 8) | (q(c) << 16) | (q(d) << 24);
    }
}

// One code as fp32.
template <bool E4M3>
__device__ __forceinline__ void codes_to_f32(uint32_t w, float (&v)[4]) {
    uint32_t lo, hi;
    codes_to_f16<E4M3>(w, lo, hi);
    v[0] = h2f(lo & 0xFFFFu);
    v[1] = h2f(lo >> 16);
    v[2] = h2f(hi & 0xFFFFu);
    v[3] = h2f(hi >> 16);
}

}  // namespace gdsllm
