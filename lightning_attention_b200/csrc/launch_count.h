// Kernels launched by this library since load, over all its files.
#pragma once

namespace lab200 {
void count_launch();  // capi.cu
}
