// logprobs_plan.hpp -- how rows of logits are cut and launched for their log
// probabilities: rules on a call's sizes, on the host and without a device.
#pragma once

#include "launch.hpp"

namespace atlas {

inline constexpr int kLogThreads = 256, kLogWaves = 4;
inline constexpr uint32_t kStrip = 1024;  // 16 logits a lane

inline uint32_t strips_of(uint32_t vocab) { return (vocab + kStrip - 1) / kStrip; }
// Two strips to a slice halve what a slice costs beside its logits; one where that
// leaves CUs idle (one row of 49152 logits 4.7 -> 4.0 us).
inline uint32_t strips_each(uint32_t rows, uint32_t vocab) { return static_cast<uint64_t>(rows) * strips_of(vocab) >= 256 * 32 ? 2 : 1; }
inline uint32_t slices_of(uint32_t rows, uint32_t vocab) {
    const uint32_t each = strips_each(rows, vocab);
    return (strips_of(vocab) + each - 1) / each;
}

// Workgroups of the first launch: a wavefront a slice, and no more than stay.
inline uint32_t sum_groups(uint32_t rows, uint32_t vocab) {
    constexpr uint32_t kGroups = 256 * 8;
    const uint64_t groups = (static_cast<uint64_t>(rows) * slices_of(rows, vocab) + kLogWaves - 1) / kLogWaves;
    return static_cast<uint32_t>(groups < kGroups ? groups : kGroups);
}

// Threads of a row's workgroup in the second: 1024 where the rows do not fill the chip
// by themselves, since its steps wait for one another and for memory (256 rows of 262144
// logits, 20 tokens each, 10 us with 256 threads).
inline uint32_t row_threads(uint32_t rows) { return rows <= 512 ? 1024 : 256; }

}  // namespace atlas
