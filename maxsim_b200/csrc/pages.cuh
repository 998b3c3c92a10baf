// Argument blocks of the page table's kernels and of the drafted trees' masks (pages.cu).
#pragma once

#include "common.cuh"

namespace msb {

// The state: page_table [sequences, max_pages], lengths [sequences], a stack of free pages and how many it has.
struct Pages {
  int32_t* table;
  int32_t* lengths;
  int32_t* free;        // [num_pages]
  int32_t* free_count;  // [1]
  int64_t num_pages;
  int sequences;
  int max_pages;
  int page_shift;
};

struct PagesExtend {
  const int32_t* tokens;  // [sequences]
  int64_t rows;
  int32_t* offsets;       // [sequences + 1]
  int64_t* slots;         // [rows]
  int32_t* positions;     // [rows]
  void* workspace;
};

constexpr int kMostTreeRows = 1024;
struct DraftTrees {
  const int32_t* parents;  // [rows], of the sequence's rows; none: the context's last token
  const int32_t* offsets;  // [batch + 1]
  int64_t rows;
  int64_t* ancestors;      // [rows, words]
  int32_t* depths;         // [rows]
  int batch;
  int max_rows;            // at most kMostTreeRows
  int words;
};

}  // namespace msb
