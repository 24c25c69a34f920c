// Element types as the kernels' launchers are told them.
#pragma once

namespace dpa {

enum DType : int { kF32 = 0, kBF16 = 1, kF16 = 2 };

}  // namespace dpa
