// How copies of pages are cut into launches: whole numbers alone, the same on the host and the device.
#pragma once

#include <cstdint>

namespace dkv {

constexpr int COPY_THREADS = 256;
// The most workgroups of a launch, which is of fewer than 2^32 work-items.
constexpr int64_t COPY_BLOCKS = ((int64_t)1 << 32) / COPY_THREADS - 1;

}  // namespace dkv
