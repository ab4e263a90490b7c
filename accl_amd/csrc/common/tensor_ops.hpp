// Tensor operators beside the collectives: the embedding of a sharded
// vocabulary with its gradient by sorted tokens, and activations kept in
// 8 bits between a forward and a backward pass. They run on the caller's
// stream (GPU) or in the calling thread (emulator ranks, whose tensors are
// host memory) and need no engine.
//
// Every function returns without waiting for the GPU; sizes and strides are
// checked by the callers and again here where a kernel's indexing rests on
// them.
#pragma once
#include "types.hpp"

namespace accl {
namespace ops {

// A token's row in this shard is id - first_row; other tokens have none.
struct EmbeddingArgs {
  const void* ids = nullptr;  // [tokens], int32 or int64
  DataType ids_dtype = DataType::int64;
  u64 tokens = 0;
  i64 first_row = 0;
  u64 rows = 0;   // of this shard
  u64 width = 0;  // of a row
  float scale = 1.0f;
  const void* src = nullptr;  // lookup: table; gradients: rows of the tokens
  i64 src_stride = 0;         // elements between rows
  DataType src_dtype = DataType::float32;
  void* dst = nullptr;  // lookup: [tokens, width]; gradient: [rows, width];
                        // sum_rows: [tokens, width]
  i64 dst_stride = 0;
  DataType dst_dtype = DataType::float32;
  bool accumulate = false;      // gradient: add to what dst holds
  void* ids_out = nullptr;      // sum_rows: [tokens], rows as ids have them
                                // less first_row, in the type of ids
  i64* count_out = nullptr;     // sum_rows: [1]
  void* workspace = nullptr;
  u64 workspace_bytes = 0;
};

// Activations kept in 8 bits. A row has `sections` equal parts whose groups
// are counted apart, so that a part can be read without its neighbour.
struct Act8Args {
  const void* x = nullptr;  // pack: source; unpack: destination
  i64 x_stride = 0;
  DataType dtype = DataType::float32;
  u64 rows = 0;
  u64 width = 0;  // of a section
  u32 sections = 1;
  signed char* codes = nullptr;  // [rows, sections * width]
  i64 codes_stride = 0;
  signed char* exps = nullptr;  // [rows, sections * groups_of(width)]
  i64 exps_stride = 0;
  // gated unit: forward writes y = silu(gate) * up, backward reads its
  // gradient there and writes the gradient of gate and up to x
  void* y = nullptr;
  i64 y_stride = 0;
};

// out[n][k] (+)= sum over rows of grad[row][n] * value[row][k]
struct WeightGradArgs {
  const void* grad = nullptr;  // [rows, outputs]
  i64 grad_stride = 0;
  DataType dtype = DataType::float32;
  u64 rows = 0;
  u64 outputs = 0;
  u64 width = 0;
  const signed char* codes = nullptr;
  i64 codes_stride = 0;
  const signed char* exps = nullptr;
  i64 exps_stride = 0;
  void* out = nullptr;  // [outputs, width]
  i64 out_stride = 0;
  DataType out_dtype = DataType::float32;
  bool accumulate = false;
  void* workspace = nullptr;
  u64 workspace_bytes = 0;
};

// GPU (gpu/embedding.hip, gpu/act8.hip, gpu/act8_wgrad.hip)
void gpu_lookup(const EmbeddingArgs& a, void* stream);
u64 gpu_gradient_workspace(u64 tokens, u64 rows, u64 width, bool to_rows);
void gpu_gradient(const EmbeddingArgs& a, void* stream);
void gpu_sum_rows(const EmbeddingArgs& a, void* stream);
void gpu_act8_pack(const Act8Args& a, void* stream);
void gpu_act8_unpack(const Act8Args& a, void* stream);
void gpu_act8_swiglu(const Act8Args& a, void* stream);
void gpu_act8_swiglu_grad(const Act8Args& a, void* stream);
u64 gpu_act8_weight_grad_workspace(const WeightGradArgs& a);
void gpu_act8_weight_grad(const WeightGradArgs& a, void* stream);

// host memory (emu/hostops.cpp)
void host_lookup(const EmbeddingArgs& a);
void host_gradient(const EmbeddingArgs& a);
void host_sum_rows(const EmbeddingArgs& a);
void host_act8_pack(const Act8Args& a);
void host_act8_unpack(const Act8Args& a);
void host_act8_swiglu(const Act8Args& a);
void host_act8_swiglu_grad(const Act8Args& a);
void host_act8_weight_grad(const WeightGradArgs& a);

}  // namespace ops
}  // namespace accl
