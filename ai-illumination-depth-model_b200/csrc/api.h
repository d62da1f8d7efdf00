// What the C entry points share: the translation of exceptions into status
// codes and the argument and CUDA checks.
#pragma once

#include <cuda_runtime.h>

#include <new>
#include <string>

#include "host.h"

#define ILL_TRY try {
#define ILL_CATCH                                          \
  }                                                        \
  catch (const Error &e) {                                 \
    set_last_error(e.what());                              \
    return e.status;                                       \
  }                                                        \
  catch (const std::bad_alloc &) {                         \
    set_last_error("out of host memory");                  \
    return ILLUMINA_INVALID_ARG;                           \
  }                                                        \
  catch (const std::exception &e) {                        \
    set_last_error(e.what());                              \
    return ILLUMINA_INVALID_ARG;                           \
  }

namespace illumina {

inline void cuda_check(cudaError_t e, const char *what) {
  if (e != cudaSuccess)
    throw Error(ILLUMINA_CUDA_ERROR, std::string(what) + ": " + cudaGetErrorName(e) + " (" + cudaGetErrorString(e) + ")");
}

inline void require(bool ok, const std::string &msg) {
  if (!ok) throw Error(ILLUMINA_INVALID_ARG, msg);
}

}  // namespace illumina
