// Device access to single elements of the paged cache (kv_layout.h).
#pragma once

#include "kv_layout.h"
#include "quant_device.h"

namespace mlq {

// Element e of position `key` of the tile at `tile` (memory or LDS), as f32.
template <int QT>
__device__ __forceinline__ float kv_element(const uint8_t* tile, int nb, bool values, int key, int e) {
    using F = KvForm<QT>;
    const int b = e >> 5, r = e & 31;
    const uint8_t* half = tile + (values ? F::half(nb) : 0);
    const uint8_t* p = half;
    int lb, lane, x;  // x: the lane's element
    if (!values) {
        lb = F::key_lane(nb);
        p += (key >> 4) * 64 * lb;
        lane = 16 * (r >> 3) + (key & 15);
        x = b * 8 + (r & 7);
    } else {
        lb = F::value_lane(nb);
        lane = 16 * ((key & 15) >> 2) + (r & 15);
        x = b * 16 + (r >> 4) * 8 + (key >> 4) * 4 + (key & 3);
    }
    if (QT == 0) return *reinterpret_cast<const float*>(p + F::at(lb, lane, 4 * x));
    float c;
    if (QT == 1) {
        c = static_cast<float>(static_cast<int>(p[F::at(lb, lane, x)]) - 128);
    } else {
        // keys: elements j and 4 + j share a byte; values: dimensions i and 16 + i
        const int byte = values ? b * 8 + (x & 7) : b * 4 + (x & 3);
        const bool high = values ? (x & 8) != 0 : (x & 4) != 0;
        const int w = p[F::at(lb, lane, byte)];
        c = static_cast<float>((high ? w >> 4 : w & 15) - (QT == 2 ? 8 : 0));
    }
    const uint16_t* scale = reinterpret_cast<const uint16_t*>(half + F::codes(nb));
    const int si = values ? F::value_scale(nb, key, b) : F::key_scale(nb, key, b);
    float y = half_value(scale[si]) * c;  // exact: 11 and at most 8 bits
    if (QT == 3) y += half_value(reinterpret_cast<const uint16_t*>(half + F::codes(nb) + F::plane(nb))[si]);
    return y;
}

}  // namespace mlq
