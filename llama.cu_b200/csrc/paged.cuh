// What the operators on a caller's pages share (paged.cu, prefix.cu).  Interface only.
#pragma once
#include "common.cuh"

namespace lcu {

int kv_pages_check(const lcu_kv_pages *p, const char *who);

}  // namespace lcu
