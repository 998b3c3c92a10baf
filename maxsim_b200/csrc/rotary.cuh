// Argument block of the rotary kernel (rotary.cu).
#pragma once

#include "common.cuh"

namespace msb {

struct Rotate {
  const void* x[2];          // queries, keys [tokens, heads, dim]; keys may be nullptr
  void* y[2];                // may be x
  int64_t x_token[2], x_head[2], y_token[2], y_head[2];  // strides in elements
  int heads[2];
  int dim;
  int half;                  // pairs that turn: dimensions past 2 half stay
  const uint64_t* turns;     // [half] turns a position, in units of 2^-64
  const uint8_t* axis;       // [half] which positions a pair goes by
  const void* positions;     // [axes, tokens], int32 or int64
  int64_t position_axis, position_token;  // strides in elements
  int wide;                  // positions are int64
  int64_t tokens;
  int neighbours;            // pairs are dimensions 2i, 2i + 1; else i, half + i
  int inverse;
  int type;
};

}  // namespace msb
