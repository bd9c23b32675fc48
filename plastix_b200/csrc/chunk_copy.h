// Which bytes of a sixteen-byte chunk are copied for a row of 16-bit values that
// starts and ends anywhere (norm.cuh, Staged). Plain C++ as well, so that the
// rule can be checked without a device.
#pragma once

#include <cstdint>

#ifdef __CUDACC__
#define PLX_CHUNK_FN __host__ __device__ __forceinline__
#else
#define PLX_CHUNK_FN inline
#endif

namespace plx {

struct ChunkCopy {
  uint32_t from, to;  // bytes of the chunk
  bool whole;         // a copy of 0 to `to` at once; else value by value
};

// The chunk at address `chunk` (a multiple of 16 that the row reaches into) of
// the row [row, row_end) of an array [begin, end): whole, with bytes of the rows
// beside it and of what lies between them, but never outside the array.
PLX_CHUNK_FN ChunkCopy chunk_copy(uint64_t chunk, uint64_t row, uint64_t row_end, uint64_t begin,
                                  uint64_t end) {
  if (chunk < begin) {  // the row's own values, which start no earlier
    const uint64_t last = row_end - chunk;
    return {(uint32_t)(row - chunk), last < 16 ? (uint32_t)last : 16u, false};
  }
  const uint64_t left = end - chunk;
  return {0u, left < 16 ? (uint32_t)left : 16u, true};
}

// Whether chunks of row r can leave an array of that many rows: others have
// eight rows, of two bytes at least each, on either side.
PLX_CHUNK_FN bool near_edge(uint32_t r, uint32_t rows) { return r < 8 || rows - r <= 8; }

}  // namespace plx
