/* Argument checks that the entry points of le_experts.cpp, le_lora.cpp and le_norm.cpp share. */
#pragma once

#include <cstdint>

#include "../../include/le_qmm.h"

static inline int le_type_bytes(int ty) { return ty == LE_F32 ? 4 : ty == LE_F16 || ty == LE_BF16 ? 2 : 0; }
static inline bool le_aligned(const void *p, unsigned n) { return ((uintptr_t)p & (n - 1)) == 0; }
