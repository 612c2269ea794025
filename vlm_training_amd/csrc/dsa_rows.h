// Eight neighbouring elements of a row in fp32, read from and written to bf16 or fp32 rows 16 bytes at a time: the element-wise kernels' currency.
#pragma once
#include "dsa_common.h"

typedef float f32x8 __attribute__((ext_vector_type(8)));

__device__ __forceinline__ f32x8 bf8_to_f32(u32x4 w) {
    f32x8 r;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        r[2 * i] = __uint_as_float(w[i] << 16);
        r[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
    return r;
}
__device__ __forceinline__ u32x4 f32_to_bf8(f32x8 x) {
    return u32x4{pack2bf(x[0], x[1]), pack2bf(x[2], x[3]), pack2bf(x[4], x[5]), pack2bf(x[6], x[7])};
}
