// qsa_io.h -- head rows of the three element types (QWFN_SRC_*) in device code.
#pragma once

#include "qsa_device.h"

namespace qwfn_qsa {

__device__ __forceinline__ float bf16_f(uint32_t h) { return __uint_as_float(h << 16); }

// Eight values of a row that begin at a 16-byte boundary.
__device__ __forceinline__ void load8(const void *p, int dtype, int64_t i, float *x) {
    if (dtype == QWFN_SRC_F32) {
        const f4v a = *reinterpret_cast<const f4v *>((const float *)p + i), b = *reinterpret_cast<const f4v *>((const float *)p + i + 4);
#pragma unroll
        for (int k = 0; k < 4; ++k) { x[k] = a[k]; x[4 + k] = b[k]; }
    } else {
        const u4v w = *reinterpret_cast<const u4v *>((const uint16_t *)p + i);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            x[2 * k] = dtype == QWFN_SRC_F16 ? h2f((uint16_t)w[k]) : bf16_f(w[k] & 0xFFFFu);
            x[2 * k + 1] = dtype == QWFN_SRC_F16 ? h2f((uint16_t)(w[k] >> 16)) : bf16_f(w[k] >> 16);
        }
    }
}

// Four values of a row at an aligned place, rounded to nearest even.
__device__ __forceinline__ void store4(void *p, int dtype, int64_t i, f4v y) {
    if (dtype == QWFN_SRC_F32) {
        *reinterpret_cast<f4v *>((float *)p + i) = y;
    } else if (dtype == QWFN_SRC_F16) {
        typedef _Float16 h4v __attribute__((ext_vector_type(4)));
        *reinterpret_cast<h4v *>((uint16_t *)p + i) = __builtin_convertvector(y, h4v);
    } else {
        typedef __bf16 b4v __attribute__((ext_vector_type(4)));
        *reinterpret_cast<b4v *>((uint16_t *)p + i) = __builtin_convertvector(y, b4v);
    }
}

// Eight of them at a 16-byte boundary.
__device__ __forceinline__ void store8(void *p, int dtype, int64_t i, const float *y) {
    if (dtype == QWFN_SRC_F32) {
        *reinterpret_cast<f4v *>((float *)p + i) = f4v{y[0], y[1], y[2], y[3]};
        *reinterpret_cast<f4v *>((float *)p + i + 4) = f4v{y[4], y[5], y[6], y[7]};
    } else if (dtype == QWFN_SRC_F16) {
        h8v h;
#pragma unroll
        for (int k = 0; k < 8; ++k) h[k] = (_Float16)y[k];
        *reinterpret_cast<h8v *>((uint16_t *)p + i) = h;
    } else {
        typedef __bf16 b8v __attribute__((ext_vector_type(8)));
        b8v h;
#pragma unroll
        for (int k = 0; k < 8; ++k) h[k] = (__bf16)y[k];
        *reinterpret_cast<b8v *>((uint16_t *)p + i) = h;
    }
}

}  // namespace qwfn_qsa
