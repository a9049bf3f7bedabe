// Sizes that the distillation loss serves, shared by the launchers and the host checks.
#pragma once

#include <stddef.h>

namespace mf {

constexpr int kDistillMostTop = 1024;             // teacher entries a row
constexpr int kDistillMostVocabulary = 3 << 17;   // one bit each in 48 KB of LDS
constexpr int kDistillMostRows = 1 << 21;         // 1024 threads a row stay below 2^32
constexpr long long kDistillMostLogits = 1ll << 35;  // (and 256 threads a part of 4096)
// (log2(e) / T and differences of logits times it stay numbers in fp32)
constexpr double kDistillLeastTemperature = 1e-6, kDistillMostTemperature = 1e6;
constexpr int kDistillStats = 4;                  // floats a row in front of its masses

// Saved for the backward pass of each row: its largest logit and the named ones' factor, the
// largest of the rest and the rest's factor, and the weighted mass of each entry.
inline size_t distill_stats_bytes(int rows, int top) {
  return sizeof(float) * (size_t)rows * (kDistillStats + top);
}

}  // namespace mf
