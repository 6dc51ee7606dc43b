// How the C ABI of the operators on nodes, hypotheses and words turns errors into codes.
#pragma once

#include <cstdint>
#include <stdexcept>
#include <string>

#include "../../include/transducer_b200.h"
#include "api_internal.h"
#include "common.cuh"

namespace tb200 {

template <typename F>
int guarded(F&& body) {
  try {
    body();
    return kOk;
  } catch (const CudaError& e) {
    return api_fail(kErrCuda, e.what());
  } catch (const std::invalid_argument& e) {
    return api_fail(kErrInvalidArgument, e.what());
  } catch (const std::exception& e) {
    return api_fail(kErrCuda, e.what());
  }
}

inline void check(bool ok, const char* what) {
  if (!ok) throw std::invalid_argument(what);
}

inline void need(size_t have, size_t want, const void* p, const char* what) {
  if (want > 0 && (p == nullptr || have < want))
    throw std::invalid_argument(std::string(what) + " too small: need " + std::to_string(want) + " bytes, got " +
                                std::to_string(have));
  if (reinterpret_cast<uintptr_t>(p) % 16 != 0)
    throw std::invalid_argument(std::string(what) + " must be 16-byte aligned");
}

}  // namespace tb200
