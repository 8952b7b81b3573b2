// Arguments of the experts' product, shared by its kernels.
#pragma once
#include "common.h"

struct ExpertArgs {
  const void *x;
  const uint8_t *packed;          // [E, R, C]
  const void *zero, *scale;       // [E, C] or [E, K / group, C]
  void *out;                      // [P, C], transposed [P, K]
  const int *order;               // [P] pairs by expert, or null: the rows of x are in that order
  const int *offsets;             // [E + 1]
  int64_t T;                      // rows of x
  int64_t P;                      // rows of the result
  int64_t R, C, group;
  int top_k, E, bits, x_dtype, zs_dtype, out_dtype, transpose;
};

// 16 rows of one expert at a time by strips of channels (expert_strip.h)
int expert_strip_f16(hipStream_t s, const ExpertArgs &a);
int expert_strip_bf16(hipStream_t s, const ExpertArgs &a);
int expert_strip_f32(hipStream_t s, const ExpertArgs &a);
// the same by tiles (expert_tile.h) of these rows x channels; K2: K in two halves, side by side
enum { TILE_32x256, TILE_64x256, TILE_64x256_K2 };
int expert_tile_f16(hipStream_t s, const ExpertArgs &a, int shape, void *ws);
int expert_tile_bf16(hipStream_t s, const ExpertArgs &a, int shape, void *ws);
int expert_tile_f32(hipStream_t s, const ExpertArgs &a, int shape, void *ws);
// the transposed product by tiles of 32, 64 or 128 rows x 256 input features (expert_back.h)
int expert_back_f16(hipStream_t s, const ExpertArgs &a, void *ws);
int expert_back_bf16(hipStream_t s, const ExpertArgs &a, void *ws);
int expert_back_f32(hipStream_t s, const ExpertArgs &a, void *ws);
