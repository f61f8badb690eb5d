// core_checks.hpp -- argument checks shared by the entry points of imq_core.h
// (core.cpp, shared.cpp).
#pragma once

#include <initializer_list>
#include <utility>

#include "core_kernels.hpp"
#include "ctx.hpp"
#include "imq_core.h"

namespace imq {
namespace detail {

// The largest element offset of a tensor walked by these extents and strides,
// or -1 where a stride is negative or the bytes pass 2^62.
inline int64_t reach(std::initializer_list<std::pair<int64_t, int64_t>> extents) {
  __int128 at = 0;
  for (const auto& e : extents) {
    if (e.second < 0) return -1;
    at += (__int128)(e.first > 0 ? e.first - 1 : 0) * e.second;
  }
  return at < ((__int128)1 << 60) ? (int64_t)at : -1;
}

// Checks *p and fills *a (core.cpp).
int check_attention(imq_ctx* ctx, const char* fn, const imq_attention_args* p, AttnArgs* a);

}  // namespace detail
}  // namespace imq
