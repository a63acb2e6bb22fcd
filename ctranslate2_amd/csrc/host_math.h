// Host-side vector sin / cos for the tables the reference builds on the CPU before a decode
// starts (sinusoidal position encodings, src/layers/common.cc:204-229; RoPE tables,
// src/layers/attention_layer.cc:252-343). The reference routes ops::Sin / ops::Cos on
// Device::CPU to Intel MKL's VML (vsSin / vsCos, src/cpu/primitives.cc:378-394) whenever it is
// built with MKL - and VML is neither libm nor correctly rounded: 4-5 % of a position table's
// entries differ from sinf / cosf by one ulp, which is enough to flip int8 activations in every
// sentence (tests/test_parity_taps_gpu.py). So the tables call the library's own entry points where an
// MKL runtime is installed (dlopen of libmkl_rt, as RCCL is; CT2X_MKL_PATH adds a search directory) and
// the C library's otherwise (NOT bit-identical to the reference). CT2X_HOST_MATH=mkl insists on the
// former, CT2X_HOST_MATH=libm on the latter.
#pragma once

#include <cstdint>

namespace ct2x {

// y[i] = sin(x[i]) / cos(x[i]) for i < n.
void host_vsin(int64_t n, const float* x, float* y);
void host_vcos(int64_t n, const float* x, float* y);
// "mkl-vml" or "libm".
const char* host_math_backend();

}  // namespace ct2x
