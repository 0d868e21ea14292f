// Low-rank adapters beside a projection: launch parameters. See kc_lora.cu.
#pragma once

#include "kc_common.cuh"

namespace kc {

constexpr int LORA_TILE = 16;      // the most rows of a tile
constexpr int LORA_MAX_RANK = 128;

// Consecutive entries of LoraParams::rows, of one adapter (-1: none).
struct LoraTile { int slot, first, n; };
struct LoraSlot { int rank; float scale; };

struct LoraParams {
  const bf16* x;             // [rows, n_in]
  const bf16* y;             // [rows, n_out]: the projection's output
  bf16* out;                 // [rows, n_out]; may be y
  const bf16* a;             // [slots][stride][n_in]
  const bf16* b;             // [slots][n_out][stride]
  const LoraSlot* slots;     // [slots]
  const LoraTile* tiles;
  const int32_t* rows;       // rows in the order of the tiles
  int n_tiles;
  int n_in, n_out;           // n_in a multiple of 32
  int stride;                // ranks kept of each adapter, those past its own zero: lora_stride(max rank)
};

// Ranks as they are stored: 16, 32, 64 or 128.
inline int lora_stride(int max_rank) {
  int r = 16;
  while (r < max_rank) r *= 2;
  return r;
}
cudaError_t lora_apply(const LoraParams& p, int sm_count, cudaStream_t s);

}  // namespace kc
