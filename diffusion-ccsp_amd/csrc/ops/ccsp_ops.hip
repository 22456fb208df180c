// libccsp_ops.so -- the operators of include/ccsp_ops.h: rows sorted by expert and combined back, the experts' products, the global gradient
// norm with clipping.  One translation unit, gfx950; the fragments below are included in order.
#include <hip/hip_runtime.h>

#include <cstdarg>
#include <cstdint>
#include <cstdio>
#include <initializer_list>
#include <type_traits>

#include "../../../include/ccsp_ops.h"

namespace {
#include "ops_common.h"
#include "ops_route.h"
#include "ops_rows.h"
#include "ops_linear.h"
#include "ops_norm.h"
}  // namespace

extern "C" {
#include "ops_abi.h"
}
