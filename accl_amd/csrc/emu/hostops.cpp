// The tensor operators on host memory, for ranks of the CPU emulator: the
// formulas as they stand, element by element, with sums in 64 bits. The
// 8-bit codes come from the same source as the GPU kernels' (common/act8.hpp),
// so a rank of either kind can read what the other kept.
#include <algorithm>
#include <cmath>
#include <numeric>
#include <vector>
#include "../common/act8.hpp"
#include "../common/arith.hpp"
#include "../common/tensor_ops.hpp"

namespace accl {
namespace ops {

// the row of the shard that token i reads, or -1
static i64 row_of(const EmbeddingArgs& a, u64 i) {
  i64 id = a.ids_dtype == DataType::int64 ? ((const i64*)a.ids)[i]
                                          : i64(((const i32*)a.ids)[i]);
  if (id < a.first_row || u64(id) - u64(a.first_row) >= a.rows) return -1;
  return i64(u64(id) - u64(a.first_row));
}

void host_lookup(const EmbeddingArgs& a) {
  for (u64 i = 0; i < a.tokens; ++i) {
    i64 r = row_of(a, i);
    for (u64 c = 0; c < a.width; ++c) {
      double v = r < 0 ? 0.0
                       : load_as_f64(a.src, u64(r * a.src_stride) + c,
                                     a.src_dtype) * double(a.scale);
      store_from_f64(a.dst, u64(i64(i) * a.dst_stride) + c, a.dst_dtype, v);
    }
  }
}

// token numbers ordered by row, and by place within a row; without the ones
// that have no row
static std::vector<u64> sorted_tokens(const EmbeddingArgs& a) {
  std::vector<u64> order;
  for (u64 i = 0; i < a.tokens; ++i)
    if (row_of(a, i) >= 0) order.push_back(i);
  std::stable_sort(order.begin(), order.end(), [&](u64 x, u64 y) {
    return row_of(a, x) < row_of(a, y);
  });
  return order;
}

// sums[c] over order[from..to)
static void sum_segment(const EmbeddingArgs& a, const std::vector<u64>& order,
                        u64 from, u64 to, std::vector<double>& sums) {
  std::fill(sums.begin(), sums.end(), 0.0);
  for (u64 j = from; j < to; ++j)
    for (u64 c = 0; c < a.width; ++c)
      sums[c] += load_as_f64(a.src, u64(i64(order[j]) * a.src_stride) + c,
                             a.src_dtype);
}

void host_gradient(const EmbeddingArgs& a) {
  std::vector<u64> order = sorted_tokens(a);
  std::vector<double> sums(a.width);
  if (!a.accumulate)
    for (u64 r = 0; r < a.rows; ++r)
      for (u64 c = 0; c < a.width; ++c)
        store_from_f64(a.dst, u64(i64(r) * a.dst_stride) + c, a.dst_dtype, 0.0);
  for (u64 j = 0; j < order.size();) {
    i64 r = row_of(a, order[j]);
    u64 end = j;
    while (end < order.size() && row_of(a, order[end]) == r) ++end;
    sum_segment(a, order, j, end, sums);
    for (u64 c = 0; c < a.width; ++c) {
      u64 at = u64(r * a.dst_stride) + c;
      double had = a.accumulate ? load_as_f64(a.dst, at, a.dst_dtype) : 0.0;
      store_from_f64(a.dst, at, a.dst_dtype,
                     had + sums[c] * double(a.scale));
    }
    j = end;
  }
}

void host_sum_rows(const EmbeddingArgs& a) {
  std::vector<u64> order = sorted_tokens(a);
  std::vector<double> sums(a.width);
  u64 count = 0;
  for (u64 j = 0; j < order.size(); ++count) {
    i64 r = row_of(a, order[j]);
    u64 end = j;
    while (end < order.size() && row_of(a, order[end]) == r) ++end;
    sum_segment(a, order, j, end, sums);
    for (u64 c = 0; c < a.width; ++c)
      store_from_f64(a.dst, u64(i64(count) * a.dst_stride) + c, a.dst_dtype,
                     sums[c] * double(a.scale));
    if (a.ids_dtype == DataType::int64) ((i64*)a.ids_out)[count] = r;
    else ((i32*)a.ids_out)[count] = i32(r);
    j = end;
  }
  for (u64 i = count; i < a.tokens; ++i) {
    for (u64 c = 0; c < a.width; ++c)
      store_from_f64(a.dst, u64(i64(i) * a.dst_stride) + c, a.dst_dtype, 0.0);
    if (a.ids_dtype == DataType::int64) ((i64*)a.ids_out)[i] = -1;
    else ((i32*)a.ids_out)[i] = -1;
  }
  *a.count_out = i64(count);
}

// ------------------------------------------------------------ 8-bit codes
static float load_float(const void* p, u64 i, DataType dt) {
  return float(load_as_f64(p, i, dt));
}

void host_act8_pack(const Act8Args& a) {
  const u64 groups = act8::groups_of(a.width);
  for (u64 r = 0; r < a.rows; ++r)
    for (u64 s = 0; s < a.sections; ++s)
      for (u64 g = 0; g < groups; ++g) {
        u64 c0 = s * a.width + g * act8::GROUP;
        u64 n = std::min<u64>(act8::GROUP, a.width - g * act8::GROUP);
        u64 at = u64(i64(r) * a.x_stride) + c0;
        u32 top = 0;
        for (u64 c = 0; c < n; ++c)
          top = std::max(top, act8::magnitude(load_float(a.x, at + c, a.dtype)));
        int e = act8::exponent_of(top);
        float inv = act8::step_inverse(e);
        for (u64 c = 0; c < n; ++c)
          a.codes[i64(r) * a.codes_stride + i64(c0 + c)] =
              e == act8::LOST
                  ? 0
                  : (signed char)act8::code_of(
                        load_float(a.x, at + c, a.dtype), inv);
        a.exps[i64(r) * a.exps_stride + i64(s * groups + g)] = (signed char)e;
      }
}

static float held(const Act8Args& a, u64 r, u64 s, u64 c) {
  int e = a.exps[i64(r) * a.exps_stride +
                 i64(s * act8::groups_of(a.width) + c / act8::GROUP)];
  if (e == act8::LOST) return NAN;
  return float(a.codes[i64(r) * a.codes_stride + i64(s * a.width + c)]) *
         act8::step(e);
}

void host_act8_unpack(const Act8Args& a) {
  for (u64 r = 0; r < a.rows; ++r)
    for (u64 s = 0; s < a.sections; ++s)
      for (u64 c = 0; c < a.width; ++c)
        store_from_f64((void*)a.x, u64(i64(r) * a.x_stride) + s * a.width + c,
                       a.dtype, double(held(a, r, s, c)));
}

void host_act8_swiglu(const Act8Args& a) {
  for (u64 r = 0; r < a.rows; ++r)
    for (u64 c = 0; c < a.width; ++c) {
      u64 at = u64(i64(r) * a.x_stride) + c;
      double gate = load_as_f64(a.x, at, a.dtype);
      double up = load_as_f64(a.x, at + a.width, a.dtype);
      store_from_f64(a.y, u64(i64(r) * a.y_stride) + c, a.dtype,
                     gate / (1.0 + std::exp(-gate)) * up);
    }
  host_act8_pack(a);
}

void host_act8_swiglu_grad(const Act8Args& a) {
  for (u64 r = 0; r < a.rows; ++r)
    for (u64 c = 0; c < a.width; ++c) {
      double gate = held(a, r, 0, c), up = held(a, r, 1, c);
      double grad = load_as_f64(a.y, u64(i64(r) * a.y_stride) + c, a.dtype);
      double sig = 1.0 / (1.0 + std::exp(-gate));
      u64 at = u64(i64(r) * a.x_stride) + c;
      store_from_f64((void*)a.x, at, a.dtype,
                     grad * up * sig * (1.0 + gate * (1.0 - sig)));
      store_from_f64((void*)a.x, at + a.width, a.dtype, grad * gate * sig);
    }
}

void host_act8_weight_grad(const WeightGradArgs& a) {
  std::vector<double> sums(a.width), x(a.width);
  // one row of the result at a time, in the order of the tokens
  for (u64 n = 0; n < a.outputs; ++n) {
    std::fill(sums.begin(), sums.end(), 0.0);
    for (u64 m = 0; m < a.rows; ++m) {
      double g = load_as_f64(a.grad, u64(i64(m) * a.grad_stride) + n, a.dtype);
      const signed char* codes = a.codes + i64(m) * a.codes_stride;
      const signed char* exps = a.exps + i64(m) * a.exps_stride;
      for (u64 k = 0; k < a.width; ++k) {
        int e = exps[k / act8::GROUP];
        if (a.dtype == DataType::float16) e = act8::exponent_in_f16(e);
        sums[k] += g * (e == act8::LOST
                            ? double(NAN)
                            : double(float(codes[k]) * act8::step(e)));
      }
    }
    for (u64 k = 0; k < a.width; ++k) {
      u64 at = u64(i64(n) * a.out_stride) + k;
      double had = a.accumulate ? load_as_f64(a.out, at, a.out_dtype) : 0.0;
      store_from_f64(a.out, at, a.out_dtype, had + sums[k]);
    }
  }
}

}  // namespace ops
}  // namespace accl
