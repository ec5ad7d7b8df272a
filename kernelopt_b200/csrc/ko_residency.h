// Which CTAs may share an SM, by the shared memory that they ask for.
//
// tcgen05.alloc waits, without a limit, until the columns that it wants are free, and a CTA of a cluster keeps its columns
// while it waits for its peers. Two kernels on two streams that met on several SMs, and wanted more than the 512 columns of
// one together, could each hold what the other waits for. So a CTA that takes more than half of the columns asks for
// kWholeTmemSmem of shared memory at least, one that takes up to half of them for kHalfTmemSmem: then whatever fits on one
// SM fits its tensor memory too, and no allocation waits for another kernel.
#pragma once

#include <cstdint>

namespace ko {

constexpr uint32_t kSmemPerSm = 228 * 1024;   // sm_100
constexpr uint32_t kSmemPerCta = 1024;        // what the system keeps for each resident CTA
constexpr uint32_t kWholeTmemSmem = 120 * 1024;
constexpr uint32_t kHalfTmemSmem = 112 * 1024;

static_assert(2 * (kWholeTmemSmem + kSmemPerCta) > kSmemPerSm, "two CTAs with all the columns");
static_assert(kWholeTmemSmem + kHalfTmemSmem + 2 * kSmemPerCta > kSmemPerSm, "one with all the columns and one with half");
static_assert(3 * (kHalfTmemSmem + kSmemPerCta) > kSmemPerSm, "three CTAs with half of the columns");
static_assert(2 * (kHalfTmemSmem + kSmemPerCta) <= kSmemPerSm, "two CTAs with half of the columns do share an SM");

}  // namespace ko
