// A launch's share of a list of tensors, passed by value: no copy to the device,
// and a captured graph keeps it.
#pragma once
#include <stdint.h>

constexpr int DES_CLIP_TENSORS = 96;

struct DesClipTable {
  const void* in[DES_CLIP_TENSORS];
  void* out[DES_CLIP_TENSORS];
  int64_t numel[DES_CLIP_TENSORS];
  int32_t first[DES_CLIP_TENSORS + 1];  // a tensor's first block; [count]: all
  uint8_t elem[DES_CLIP_TENSORS];       // des::Elem
  int32_t count;
};
