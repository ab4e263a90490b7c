// Python bindings of the tensor operators (common/tensor_ops.hpp). Operands
// come as addresses, as those of call_raw do; accl_amd/torch_ops.py checks
// the tensors behind them. `stream` is the caller's HIP stream, or -1 for
// operands in host memory.
#include <pybind11/pybind11.h>
#include "../common/tensor_ops.hpp"
#include "../core/util.hpp"
#include "tensor_ops.hpp"

namespace py = pybind11;
using namespace accl;

static ops::EmbeddingArgs embedding_args(u64 ids, u32 ids_dtype, u64 tokens,
                                         i64 first_row, u64 rows, u64 width,
                                         float scale, u64 src, i64 src_stride,
                                         u32 src_dtype, u64 dst, i64 dst_stride,
                                         u32 dst_dtype) {
  ops::EmbeddingArgs a;
  a.ids = (const void*)ids;
  a.ids_dtype = DataType(ids_dtype);
  a.tokens = tokens;
  a.first_row = first_row;
  a.rows = rows;
  a.width = width;
  a.scale = scale;
  a.src = (const void*)src;
  a.src_stride = src_stride;
  a.src_dtype = DataType(src_dtype);
  a.dst = (void*)dst;
  a.dst_stride = dst_stride;
  a.dst_dtype = DataType(dst_dtype);
  return a;
}

static ops::Act8Args act8_args(u64 x, i64 x_stride, u32 dtype, u64 rows,
                               u64 width, u32 sections, u64 codes,
                               i64 codes_stride, u64 exps, i64 exps_stride,
                               u64 y, i64 y_stride) {
  ops::Act8Args a;
  a.x = (const void*)x;
  a.x_stride = x_stride;
  a.dtype = DataType(dtype);
  a.rows = rows;
  a.width = width;
  a.sections = sections;
  a.codes = (signed char*)codes;
  a.codes_stride = codes_stride;
  a.exps = (signed char*)exps;
  a.exps_stride = exps_stride;
  a.y = (void*)y;
  a.y_stride = y_stride;
  return a;
}

void register_tensor_ops(py::module_& m) {
  m.def("ops_lookup",
        [](i64 stream, u64 ids, u32 ids_dtype, u64 tokens, i64 first_row,
           u64 rows, u64 width, float scale, u64 src, i64 src_stride,
           u32 src_dtype, u64 dst, i64 dst_stride, u32 dst_dtype) {
          auto a = embedding_args(ids, ids_dtype, tokens, first_row, rows,
                                  width, scale, src, src_stride, src_dtype,
                                  dst, dst_stride, dst_dtype);
          if (stream < 0) ops::host_lookup(a);
          else ops::gpu_lookup(a, (void*)stream);
        });
  m.def("ops_gradient_workspace", &ops::gpu_gradient_workspace);
  m.def("ops_gradient",
        [](i64 stream, u64 ids, u32 ids_dtype, u64 tokens, i64 first_row,
           u64 rows, u64 width, float scale, u64 src, i64 src_stride,
           u32 src_dtype, u64 dst, i64 dst_stride, u32 dst_dtype,
           bool accumulate, u64 workspace, u64 workspace_bytes) {
          auto a = embedding_args(ids, ids_dtype, tokens, first_row, rows,
                                  width, scale, src, src_stride, src_dtype,
                                  dst, dst_stride, dst_dtype);
          a.accumulate = accumulate;
          a.workspace = (void*)workspace;
          a.workspace_bytes = workspace_bytes;
          if (stream < 0) ops::host_gradient(a);
          else ops::gpu_gradient(a, (void*)stream);
        });
  m.def("ops_sum_rows",
        [](i64 stream, u64 ids, u32 ids_dtype, u64 tokens, i64 first_row,
           u64 rows, u64 width, float scale, u64 src, i64 src_stride,
           u32 src_dtype, u64 dst, i64 dst_stride, u32 dst_dtype, u64 ids_out,
           u64 count_out, u64 workspace, u64 workspace_bytes) {
          auto a = embedding_args(ids, ids_dtype, tokens, first_row, rows,
                                  width, scale, src, src_stride, src_dtype,
                                  dst, dst_stride, dst_dtype);
          a.ids_out = (void*)ids_out;
          a.count_out = (i64*)count_out;
          a.workspace = (void*)workspace;
          a.workspace_bytes = workspace_bytes;
          if (stream < 0) ops::host_sum_rows(a);
          else ops::gpu_sum_rows(a, (void*)stream);
        });
  m.def("ops_act8_pack",
        [](i64 stream, u64 x, i64 x_stride, u32 dtype, u64 rows, u64 width,
           u32 sections, u64 codes, i64 codes_stride, u64 exps,
           i64 exps_stride) {
          auto a = act8_args(x, x_stride, dtype, rows, width, sections, codes,
                             codes_stride, exps, exps_stride, 0, 0);
          if (stream < 0) ops::host_act8_pack(a);
          else ops::gpu_act8_pack(a, (void*)stream);
        });
  m.def("ops_act8_unpack",
        [](i64 stream, u64 x, i64 x_stride, u32 dtype, u64 rows, u64 width,
           u32 sections, u64 codes, i64 codes_stride, u64 exps,
           i64 exps_stride) {
          auto a = act8_args(x, x_stride, dtype, rows, width, sections, codes,
                             codes_stride, exps, exps_stride, 0, 0);
          if (stream < 0) ops::host_act8_unpack(a);
          else ops::gpu_act8_unpack(a, (void*)stream);
        });
  // width: of one half of x
  m.def("ops_act8_swiglu",
        [](i64 stream, u64 x, i64 x_stride, u32 dtype, u64 rows, u64 width,
           u64 codes, i64 codes_stride, u64 exps, i64 exps_stride, u64 y,
           i64 y_stride) {
          auto a = act8_args(x, x_stride, dtype, rows, width, 2, codes,
                             codes_stride, exps, exps_stride, y, y_stride);
          if (stream < 0) ops::host_act8_swiglu(a);
          else ops::gpu_act8_swiglu(a, (void*)stream);
        });
  m.def("ops_act8_swiglu_grad",
        [](i64 stream, u64 x, i64 x_stride, u32 dtype, u64 rows, u64 width,
           u64 codes, i64 codes_stride, u64 exps, i64 exps_stride, u64 y,
           i64 y_stride) {
          auto a = act8_args(x, x_stride, dtype, rows, width, 2, codes,
                             codes_stride, exps, exps_stride, y, y_stride);
          if (stream < 0) ops::host_act8_swiglu_grad(a);
          else ops::gpu_act8_swiglu_grad(a, (void*)stream);
        });
  m.def("ops_act8_weight_grad_workspace",
        [](u64 grad, i64 grad_stride, u32 dtype, u64 rows, u64 outputs,
           u64 width) {
          ops::WeightGradArgs a;
          a.grad = (const void*)grad;
          a.grad_stride = grad_stride;
          a.dtype = DataType(dtype);
          a.rows = rows;
          a.outputs = outputs;
          a.width = width;
          return ops::gpu_act8_weight_grad_workspace(a);
        });
  m.def("ops_act8_weight_grad",
        [](i64 stream, u64 grad, i64 grad_stride, u32 dtype, u64 rows,
           u64 outputs, u64 width, u64 codes, i64 codes_stride, u64 exps,
           i64 exps_stride, u64 out, i64 out_stride, u32 out_dtype,
           bool accumulate, u64 workspace, u64 workspace_bytes) {
          ops::WeightGradArgs a;
          a.grad = (const void*)grad;
          a.grad_stride = grad_stride;
          a.dtype = DataType(dtype);
          a.rows = rows;
          a.outputs = outputs;
          a.width = width;
          a.codes = (const signed char*)codes;
          a.codes_stride = codes_stride;
          a.exps = (const signed char*)exps;
          a.exps_stride = exps_stride;
          a.out = (void*)out;
          a.out_stride = out_stride;
          a.out_dtype = DataType(out_dtype);
          a.accumulate = accumulate;
          a.workspace = (void*)workspace;
          a.workspace_bytes = workspace_bytes;
          if (stream < 0) ops::host_act8_weight_grad(a);
          else ops::gpu_act8_weight_grad(a, (void*)stream);
        });
}
