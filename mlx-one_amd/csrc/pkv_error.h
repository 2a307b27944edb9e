// pkv_error.h -- error reporting shared by the extern "C" entry points.
#pragma once
#include <hip/hip_runtime.h>

#include <string>

#include "pkv.h"
#include "pkv_format.h"

namespace pkv {

// Records the calling thread's error text (pkv_last_error) and returns `code`.
int fail(int code, const std::string &message);
int check_launch(hipError_t e, const char *what);
// The layout's sizes; an error code for layouts that do not exist.
int geometry(const pkv_layout *layout, pkv_geometry *g);

}  // namespace pkv
