// Sizes that the norms serve, shared by the launchers and the host checks.
#pragma once

namespace mf {

constexpr int kNormMostVectors = 8;     // 16-byte vectors of a row that a lane holds
constexpr int kNormMostDim = 16384;     // 512 lanes of 8 fp32 vectors
constexpr int kNormMostRows = 1 << 22;  // 512 lanes a row stay below 2^32 threads

constexpr int kNormFewRows = 1024;      // rows whose weights' gradients take no second launch

}  // namespace mf
