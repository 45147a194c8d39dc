// Pages of a KV cache: what the kernels and the pool share.
#pragma once

#include "dmath.h"
#include "rt.h"

// One layer's pages on the device: bf16 [n_pages, Hkv, R, hd] each, R = 2^shift rows a page.
struct KvLayer {
  bf16_t* k;
  bf16_t* v;
  int n_pages, Hkv, shift;
};

// Host checks that every entry point over pages makes (before anything of the context is touched).
int kv_pages_check(const ornith_kv_pages* p, const char* who);
int kv_batch_check(const ornith_kv_pages* p, const ornith_kv_batch* b, const char* who);

static inline int kv_shift(int page_rows) { return __builtin_ctz((unsigned)page_rows); }
static inline KvLayer kv_layer(const ornith_kv_pages* p, int layer) {
  return KvLayer{static_cast<bf16_t*>(p->d_k[layer]), static_cast<bf16_t*>(p->d_v[layer]), p->n_pages, p->Hkv, kv_shift(p->page_rows)};
}
