/* What the entry points outside le_qmm.cpp use of a context, whose definition lives there. None of these lets a C++
 * exception out. */
#pragma once

#include <hip/hip_runtime.h>

#include <cstddef>

#include "../../include/le_qmm.h"

int le_ctx_device(const le_ctx *ctx);
int le_ctx_cus(const le_ctx *ctx); /* compute units of the context's device */
/* Sets the context's error text and returns code. */
int le_ctx_fail(le_ctx *ctx, int code, const char *msg);
int le_ctx_failf(le_ctx *ctx, int code, const char *fmt, ...) __attribute__((format(printf, 3, 4)));
/* LE_OK where the calling thread's current device is the context's (its kernels are loaded there), else LE_ERR_ARG. */
int le_ctx_on_device(le_ctx *ctx);
int le_ctx_launch(le_ctx *ctx, const char *name, dim3 grid, int block, size_t lds, hipStream_t st, void **args);
