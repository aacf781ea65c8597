// Host interface of the tcgen05 kernels over the 8-bit paged KV cache.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include "paged8.cuh"

namespace vo {

// pages that 128-key tiles can be staged from: they divide the tile or are a multiple of it, in whole 8-row groups, and
// the pool's rows fit the copies' 32-bit coordinates
inline bool paged8_pages_ok(const p8::AttendArgs& a) {
  const bool fits = a.block <= 128 ? a.block >= 8 && 128 % a.block == 0 : a.block % 128 == 0;
  return fits && (int64_t)a.pages * a.Hk * a.block < (1ll << 31) - 128;
}

// few query rows (tokens x heads of a group <= 16)
bool paged8_decode_ok(const p8::AttendArgs& a);
int64_t paged8_decode_workspace(const p8::AttendArgs& a, int sms);  // bytes
int paged8_decode_launch(const p8::AttendArgs& a, void* workspace, int sms, cudaStream_t stream, int* launches);
int paged8_decode_error(bool reset);

// any number of query rows
bool paged8_chunk_ok(const p8::AttendArgs& a);
int64_t paged8_chunk_workspace(const p8::AttendArgs& a, int sms);
int paged8_chunk_launch(const p8::AttendArgs& a, void* workspace, int sms, cudaStream_t stream, int* launches);
int paged8_chunk_error(bool reset);

}  // namespace vo
