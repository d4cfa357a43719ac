// Launch wrappers of the adapter kernels, shared with their C ABI
// (include/nkt_lora.h).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace nkt {

// One projection's adapters as the kernels address them (layouts in
// include/nkt_lora.h).
struct LoraView {
  const uint16_t* a;
  const uint16_t* b;
  const float* scales;
  const int32_t* ranks;
  uint32_t* status;
  int adapters, parts, in, columns;
  int rank;         // padded: 16, 32, 64 or 128
  int row_blocks;   // of 32 rows of A
  int part_end[4];  // blocks of 64 columns up to and with each part
};

struct LoraArgs {
  const uint16_t* x;
  const uint16_t* base;
  uint16_t* out;
  int64_t x_stride, base_stride, out_stride;
  const int64_t* index;
  int tokens;
  // workspace, where tokens are grouped by adapter
  uint16_t* low;          // scale * x A^T as operands: [tiles of 32 tokens, parts, R / 16, 2, 2, 32, 8]
  int32_t* order;         // [tiles, 32] tokens, -1: none
  int32_t* tile_adapter;  // [tiles]
};

size_t lora_workspace_bytes(const LoraView& v, int tokens);
hipError_t launch_lora(const LoraView& v, LoraArgs a, void* workspace, hipStream_t stream);

}  // namespace nkt
