/* SPDX-License-Identifier: Apache-2.0 */
/* dsv4_elem.h - activations in one of three element types (DSV4_HIP_F32,
 * DSV4_HIP_BF16, DSV4_HIP_F16) as fp32 values in registers: whole 16-byte
 * vectors where rows allow it, single elements elsewhere. Values widen
 * exactly; narrowing rounds once, to nearest even. */
#ifndef DSV4_ELEM_H
#define DSV4_ELEM_H

#include "dsv4_dev.h"
#include "../../include/dsv4_hip.h"

namespace dsv4 {

template <int TYPE> constexpr int elem_bytes() { return TYPE == DSV4_HIP_F32 ? 4 : 2; }
static inline int elem_bytes_of(int type) { return type == DSV4_HIP_F32 ? 4 : 2; }

__device__ __forceinline__ uint32_t bf16_bits(float f)
{
    const uint32_t u = __float_as_uint(f);
    if ((u & 0x7FFFFFFFu) > 0x7F800000u) return (u >> 16) | 0x40u;   /* quiet NaN */
    return (u + 0x7FFFu + ((u >> 16) & 1u)) >> 16;
}

/* one 16-bit element in the low half of u */
template <int TYPE>
__device__ __forceinline__ float widen16(uint32_t u)
{
    if constexpr (TYPE == DSV4_HIP_BF16) return __uint_as_float(u << 16);
    else return (float)__builtin_bit_cast(_Float16, (uint16_t)u);
}
template <int TYPE>
__device__ __forceinline__ uint32_t narrow16(float f)
{
    if constexpr (TYPE == DSV4_HIP_BF16) return bf16_bits(f);
    else return __builtin_bit_cast(uint16_t, (_Float16)f);
}

/* V elements from p: a whole 16-byte vector (V = 4 fp32 or 8 of 16 bits) or
 * one element (V = 1) */
template <int TYPE, int V>
struct Elem {
    static_assert(V == 1 || V * elem_bytes<TYPE>() == 16, "one element or a whole vector");
    u32x4 raw;
    /* ONCE: bytes that the call reads once and that no cache should keep */
    template <bool ONCE = false>
    __device__ __forceinline__ void load(const void *p)
    {
        if constexpr (V > 1 && ONCE) raw = __builtin_nontemporal_load(gptr((const u32x4 *)p));
        else if constexpr (V > 1) raw = *gptr((const u32x4 *)p);
        else if constexpr (TYPE == DSV4_HIP_F32) raw.x = *gptr((const uint32_t *)p);
        else raw.x = *gptr((const uint16_t *)p);
    }
    __device__ __forceinline__ void store(void *p) const
    {
        if constexpr (V > 1) *(DSV4_GLOBAL u32x4 *)p = raw;
        else if constexpr (TYPE == DSV4_HIP_F32) *(DSV4_GLOBAL uint32_t *)p = raw.x;
        else *(DSV4_GLOBAL uint16_t *)p = (uint16_t)raw.x;
    }
    __device__ __forceinline__ void get(float (&f)[V]) const
    {
        if constexpr (TYPE == DSV4_HIP_F32) {
#pragma unroll
            for (int i = 0; i < V; i++) f[i] = __uint_as_float(raw[i]);
        } else if constexpr (V == 1) {
            f[0] = widen16<TYPE>(raw.x);
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++) {
                f[2 * i] = widen16<TYPE>(raw[i] & 0xFFFFu);
                f[2 * i + 1] = widen16<TYPE>(raw[i] >> 16);
            }
        }
    }
    __device__ __forceinline__ void set(const float (&f)[V])
    {
        if constexpr (TYPE == DSV4_HIP_F32) {
#pragma unroll
            for (int i = 0; i < V; i++) raw[i] = __float_as_uint(f[i]);
        } else if constexpr (V == 1) {
            raw.x = narrow16<TYPE>(f[0]);
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++) raw[i] = narrow16<TYPE>(f[2 * i]) | (narrow16<TYPE>(f[2 * i + 1]) << 16);
        }
    }
};

} // namespace dsv4

#endif /* DSV4_ELEM_H */
