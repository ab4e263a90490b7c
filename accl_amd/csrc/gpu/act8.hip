// Activations kept in 8 bits (common/act8.hpp): packing, reading back, and
// the gated unit y = silu(gate) * up whose inputs are kept that way.
//
// Every kernel is one pass over memory, and that is what bounds it: for bf16
// packing 16384 x 8192 takes 75 us (5.4 TB/s, where a large copy reaches 4.9),
// unpacking 70 us (5.8); the gated unit of 8192 x 12288 131 us forward (6.2) and
// 145 us backward (5.6). A lane holds eight neighbouring values, so four lanes
// share a group and find its largest magnitude with two exchanges inside a quad
// of lanes. Values go out past the caches, since what is kept or handed on is
// larger than they are (pack and unpack: 159 us into the caches, 152 past them);
// codes do not (143 and 155).
#include <hip/hip_runtime.h>
#include "../common/act8.hpp"
#include "../common/tensor_ops.hpp"
#include "ops_device.hpp"

namespace accl {
namespace ops {

constexpr int QUAD_SWAP_1 = 0xB1;  // lanes 1 0 3 2
constexpr int QUAD_SWAP_2 = 0x4E;  // lanes 2 3 0 1

__device__ inline u32 quad_max(u32 v) {
  u32 o = u32(__builtin_amdgcn_mov_dpp(int(v), QUAD_SWAP_1, 0xF, 0xF, true));
  v = v > o ? v : o;
  o = u32(__builtin_amdgcn_mov_dpp(int(v), QUAD_SWAP_2, 0xF, 0xF, true));
  return v > o ? v : o;
}

// Codes of a lane's eight values and its group's exponent; every lane of the
// quad calls it.
template <class T>
__device__ inline int pack8(const Eight<T>& v, u32x2& codes) {
  u32 top = 0;
#pragma unroll
  for (int i = 0; i < VEC; ++i) {
    const u32 m = act8::magnitude(float(v.e[i]));
    top = top > m ? top : m;
  }
  const int e = act8::exponent_of(quad_max(top));
  const float inv = act8::step_inverse(e), most = 127.0f * act8::step(e);
  // x / 2^e is exact, so that cutting x first changes nothing; 1.5 * 2^23 added
  // to it rounds it to a whole number, whose low byte is the code
  u32 word[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    u32 b[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      b[i] = act8::float_bits(__builtin_fmaf(
          __builtin_amdgcn_fmed3f(float(v.e[h * 4 + i]), -most, most), inv,
          12582912.0f));
    word[h] = __builtin_amdgcn_perm(__builtin_amdgcn_perm(b[3], b[2], 0x0C0C0400),
                                    __builtin_amdgcn_perm(b[1], b[0], 0x0C0C0400),
                                    0x05040100);
  }
  codes.x = e == act8::LOST ? 0 : word[0];
  codes.y = e == act8::LOST ? 0 : word[1];
  return e;
}

__device__ inline void store_codes(signed char* p, int n, u32x2 codes) {
  if (n >= VEC) {
    *(u32x2_any*)p = codes;
  } else {
#pragma unroll
    for (int i = 0; i < VEC; ++i)
      if (i < n) p[i] = (signed char)(codes[i / 4] >> (8 * (i % 4)));
  }
}

__device__ inline u32x2 load_codes(const signed char* p, int n) {
  if (n >= VEC) return *(const u32x2_any*)p;
  u32 word[2] = {0, 0};
#pragma unroll
  for (int i = 0; i < VEC; ++i)
    if (i < n) word[i / 4] |= u32((unsigned char)p[i]) << (8 * (i % 4));
  return u32x2{word[0], word[1]};
}

// What the codes stand for; a lost group gives NaN.
__device__ inline void held8(u32x2 codes, int e, float v[VEC]) {
  const float step = e == act8::LOST ? __builtin_nanf("") : act8::step(e);
#pragma unroll
  for (int i = 0; i < VEC; ++i)
    v[i] = float((signed char)(codes[i / 4] >> (8 * (i % 4)))) * step;
}

// A wave's place: SPAN columns of a section; n is how many are this lane's.
struct Place {
  u64 section, c;
  int n;
  __device__ Place(u64 width) {
    const u32 spans = u32((width + SPAN - 1) / SPAN);
    section = blockIdx.x / spans;
    c = u64(blockIdx.x % spans) * SPAN + (threadIdx.x & 63) * VEC;
    n = c < width ? int(width - c < VEC ? width - c : VEC) : 0;
  }
};

template <class T>
__global__ void __launch_bounds__(256) pack_kernel(Act8Args a) {
  const Place at(a.width);
  const i64 groups = i64(act8::groups_of(a.width));
  for (u64 r = u64(blockIdx.y) * 4 + (threadIdx.x >> 6); r < a.rows;
       r += u64(gridDim.y) * 4) {
    const i64 col = i64(at.section * a.width + at.c);
    Eight<T> v;
    load8((const T*)a.x + i64(r) * a.x_stride + col, at.n, v);
    u32x2 codes;
    const int e = pack8(v, codes);
    if (at.n == 0) continue;
    store_codes(a.codes + i64(r) * a.codes_stride + col, at.n, codes);
    if (at.c % act8::GROUP == 0)
      a.exps[i64(r) * a.exps_stride + i64(at.section) * groups +
             i64(at.c / act8::GROUP)] = (signed char)e;
  }
}

template <class T>
__global__ void __launch_bounds__(256) unpack_kernel(Act8Args a) {
  const Place at(a.width);
  const i64 groups = i64(act8::groups_of(a.width));
  if (at.n == 0) return;
  for (u64 r = u64(blockIdx.y) * 4 + (threadIdx.x >> 6); r < a.rows;
       r += u64(gridDim.y) * 4) {
    const i64 col = i64(at.section * a.width + at.c);
    float f[VEC];
    held8(load_codes(a.codes + i64(r) * a.codes_stride + col, at.n),
          a.exps[i64(r) * a.exps_stride + i64(at.section) * groups +
                 i64(at.c / act8::GROUP)],
          f);
    Eight<T> v;
#pragma unroll
    for (int i = 0; i < VEC; ++i) v.e[i] = T(f[i]);
    stream8((T*)a.x + i64(r) * a.x_stride + col, at.n, v);
  }
}

// 1 / (1 + exp(-x)) for a result in T. For float32 it is off by at most 7 units of
// 2^-24 of its size: two of the power, one each of its factor, their product and
// the sum, two of the reciprocal. The factor is what rounding x log2(e) left, which
// goes into the exponent: without it, as for the 16-bit types, the result is off
// by up to |x| units more, of which their rounding shows none (and the gradient of
// 8192 x 12288 bf16 takes 135 us instead of 141).
template <class T>
__device__ inline float logistic(float x) {
  if constexpr (sizeof(T) == 2) {
    return __builtin_amdgcn_rcpf(1.0f + __expf(-x));
  } else {
    // REST: log2(e) - LOG2E
    constexpr float LOG2E = 0x1.715476p+0f, REST = 0x1.4ae0cp-26f;
    constexpr float LN2 = 0x1.62e43p-1f;
    const float v = __builtin_amdgcn_fmed3f(-x, -128.0f, 128.0f);
    const float t = v * LOG2E;
    const float left = __builtin_fmaf(v, REST, __builtin_fmaf(v, LOG2E, -t));
    const float e =
        __builtin_amdgcn_exp2f(t) * __builtin_fmaf(left, LN2, 1.0f);
    return __builtin_amdgcn_rcpf(1.0f + e);
  }
}

template <class T>
__global__ void __launch_bounds__(256) swiglu_kernel(Act8Args a) {
  const Place at(a.width);
  const i64 groups = i64(act8::groups_of(a.width));
  for (u64 r = u64(blockIdx.y) * 4 + (threadIdx.x >> 6); r < a.rows;
       r += u64(gridDim.y) * 4) {
    const T* x = (const T*)a.x + i64(r) * a.x_stride + i64(at.c);
    Eight<T> gate, up, y;
    load8(x, at.n, gate);
    load8(x + a.width, at.n, up);
    u32x2 gate_codes, up_codes;
    const int gate_e = pack8(gate, gate_codes), up_e = pack8(up, up_codes);
    if (at.n == 0) continue;
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      const float g = float(gate.e[i]);
      y.e[i] = T(g * logistic<T>(g) * float(up.e[i]));
    }
    stream8((T*)a.y + i64(r) * a.y_stride + i64(at.c), at.n, y);
    signed char* codes = a.codes + i64(r) * a.codes_stride + i64(at.c);
    store_codes(codes, at.n, gate_codes);
    store_codes(codes + a.width, at.n, up_codes);
    if (at.c % act8::GROUP == 0) {
      signed char* e = a.exps + i64(r) * a.exps_stride + at.c / act8::GROUP;
      e[0] = (signed char)gate_e;
      e[groups] = (signed char)up_e;
    }
  }
}

// d gate = grad up s (1 + gate (1 - s)), d up = grad gate s, s = logistic(gate)
template <class T>
__global__ void __launch_bounds__(256) swiglu_grad_kernel(Act8Args a) {
  const Place at(a.width);
  const i64 groups = i64(act8::groups_of(a.width));
  if (at.n == 0) return;
  for (u64 r = u64(blockIdx.y) * 4 + (threadIdx.x >> 6); r < a.rows;
       r += u64(gridDim.y) * 4) {
    const signed char* codes = a.codes + i64(r) * a.codes_stride + i64(at.c);
    const signed char* e = a.exps + i64(r) * a.exps_stride + at.c / act8::GROUP;
    float gate[VEC], up[VEC];
    held8(load_codes(codes, at.n), e[0], gate);
    held8(load_codes(codes + a.width, at.n), e[groups], up);
    Eight<T> grad, d_gate, d_up;
    load8((const T*)a.y + i64(r) * a.y_stride + i64(at.c), at.n, grad);
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      const float d = float(grad.e[i]), s = logistic<T>(gate[i]);
      d_gate.e[i] = T(d * up[i] * s * (1.0f + gate[i] * (1.0f - s)));
      d_up.e[i] = T(d * gate[i] * s);
    }
    T* x = (T*)a.x + i64(r) * a.x_stride + i64(at.c);
    stream8(x, at.n, d_gate);
    stream8(x + a.width, at.n, d_up);
  }
}

static dim3 grid_of(const Act8Args& a, u32 sections) {
  return dim3(sections * blocks_of(a.width, SPAN),
              u32(a.rows / 4 < 65535 ? (a.rows + 3) / 4 : 65535));
}

#define ACCL_ACT8_LAUNCH(fn, kernel, what, sections)                        \
  void fn(const Act8Args& a, void* stream) {                                \
    if (!a.rows || !a.width) return;                                        \
    with_type(a.dtype, what, [&](auto t) {                                  \
      using T = decltype(t);                                                \
      hipLaunchKernelGGL((kernel<T>), grid_of(a, sections), dim3(256), 0,   \
                         (hipStream_t)stream, a);                           \
    });                                                                     \
    launched(what);                                                         \
  }

ACCL_ACT8_LAUNCH(gpu_act8_pack, pack_kernel, "act8_pack", a.sections)
ACCL_ACT8_LAUNCH(gpu_act8_unpack, unpack_kernel, "act8_unpack", a.sections)
ACCL_ACT8_LAUNCH(gpu_act8_swiglu, swiglu_kernel, "act8_swiglu", 1)
ACCL_ACT8_LAUNCH(gpu_act8_swiglu_grad, swiglu_grad_kernel, "act8_swiglu_grad", 1)

}  // namespace ops
}  // namespace accl
