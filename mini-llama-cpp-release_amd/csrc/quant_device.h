// What the device's block quantizers share: the reference's binary16 rounding of
// scales and the fold of a quad of lanes (quantize.hip, kv_cache.hip).
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace mlq {

__device__ __forceinline__ uint32_t f32_bits(float v) { return __builtin_bit_cast(uint32_t, v); }

// f32 -> binary16 with the reference's rounding (round half up
// in magnitude at the first dropped bit, overflow and NaN to Inf, src/quant.cpp:19-55).
__device__ __forceinline__ uint16_t half_round_up(float value) {
    const uint32_t u = f32_bits(value);
    const uint32_t sign = (u >> 16) & 0x8000u;
    const int e = static_cast<int>((u >> 23) & 0xffu) - 112;
    const uint32_t frac = u & 0x7fffffu;
    if (e >= 31) return static_cast<uint16_t>(sign | 0x7c00u);
    if (e <= 0) {
        if (e < -10) return static_cast<uint16_t>(sign);
        uint32_t sig = (frac | 0x800000u) >> (1 - e);
        sig += (sig & 0x1000u) << 1;  // +0x2000 when the first dropped bit is set
        return static_cast<uint16_t>(sign | (sig >> 13));
    }
    uint32_t sig = frac + ((frac & 0x1000u) << 1);
    int eh = e;
    if (sig & 0x800000u) {
        sig = 0;
        if (++eh >= 31) return static_cast<uint16_t>(sign | 0x7c00u);
    }
    return static_cast<uint16_t>(sign | (static_cast<uint32_t>(eh) << 10) | (sig >> 13));
}

__device__ __forceinline__ float half_value(uint16_t h) {
    return (float)__builtin_bit_cast(_Float16, h);  // exact (v_cvt_f32_f16)
}

__device__ __forceinline__ int round_int(float v) { return static_cast<int>(roundf(v)); }

// The other lane of the quad that differs in bit 0 (CTRL 0xB1) or bit 1 (0x4E).
template <int CTRL>
__device__ __forceinline__ float quad_peer(float v) {
    return __builtin_bit_cast(
        float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}

// Largest of a quad's values (none is NaN).
__device__ __forceinline__ float quad_max(float v) {
    float o = quad_peer<0xB1>(v);
    v = (v < o) ? o : v;
    o = quad_peer<0x4E>(v);
    return (v < o) ? o : v;
}

// Smallest of a quad's values (none is NaN); of equal ones the lowest lane's, as a
// scan in element order keeps it (it decides the sign of a zero).
__device__ __forceinline__ float quad_first_min(float v, int l) {
    float o = quad_peer<0xB1>(v);
    v = (l & 1) ? ((v < o) ? v : o) : ((o < v) ? o : v);
    o = quad_peer<0x4E>(v);
    return (l & 2) ? ((v < o) ? v : o) : ((o < v) ? o : v);
}

}  // namespace mlq
