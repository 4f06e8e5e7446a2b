// The checks of a packed cache's descriptor.
#pragma once
#include "entry.cuh"

namespace ocrvl {

inline int check_packed(const ocrvl_packed_cache *c) {
  if (!c) return invalid("null cache");
  if (c->head_dim != 64 && c->head_dim != 128) return invalid("head_dim must be 64 or 128");
  if (c->num_kv_heads < 1 || c->num_layers < 1 || c->batch < 1 || c->max_pages < 1 || c->num_pages < 1)
    return invalid("cache dimensions must be positive");
  if (c->batch > 65535) return invalid("at most 65535 sequences a call");
  if (c->page_size < 16 || c->page_size & (c->page_size - 1)) return invalid("page_size must be a power of two of at least 16");
  if ((long long)c->max_pages * c->page_size > 0x40000000ll) return invalid("at most 2^30 positions a sequence");
  if (c->reserved) return invalid("reserved must be 0");
  if (!c->k || !c->v || !c->k_scale || !c->v_scale || !c->table) return invalid("null cache pointer");
  if (!aligned16(c->k) || !aligned16(c->v) || !aligned16(c->k_scale) || !aligned16(c->v_scale))
    return invalid("k, v and their scales must be 16-byte aligned");
  for (long long s : {c->page_stride, c->layer_stride, c->head_stride})
    if (s < 0 || s % 16) return invalid("strides of the codes must be non-negative multiples of 16 bytes");
  for (long long s : {c->scale_page_stride, c->scale_layer_stride, c->scale_head_stride})
    if (s < 0 || s % 8) return invalid("strides of the scales must be non-negative multiples of 16 bytes");
  if (c->table_stride < (c->batch > 1 ? c->max_pages : 0)) return invalid("table_stride is shorter than a row");
  return OCRVL_OK;
}

}  // namespace ocrvl
