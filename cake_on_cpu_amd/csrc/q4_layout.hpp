// q4_layout.hpp -- the packed form of 4-bit weights (described in q4_kernels.hip) and the choice of
// a kernel's instance by element type and group size.
#pragma once

#include <hip/hip_runtime.h>

#include <cstddef>
#include <type_traits>

#include "cake_hip.h"

namespace cake {

struct Q4Layout {
    int N, K;
    int tiles, blocks;          // ceil(N / 16), ceil(K / 128)
    int groups_per_block;       // 128 / group: 1, 2 or 4
    int scale_type;             // CAKE_HIP_F32, _F16 or _BF16
    size_t scales_at, zeros_at; // byte offsets behind the codes
    size_t bytes;
};
Q4Layout q4_layout(int N, int K, int group, int scale_type, bool with_zeros);

template <class F>
void q4_for_type_and_group(int type, int groups_per_block, F&& go)
{
    auto with_group = [&](auto t) {
        if (groups_per_block == 1) go(t, std::integral_constant<int, 1>());
        else if (groups_per_block == 2) go(t, std::integral_constant<int, 2>());
        else go(t, std::integral_constant<int, 4>());
    };
    if (type == CAKE_HIP_F32) with_group(std::integral_constant<int, CAKE_HIP_F32>());
    else if (type == CAKE_HIP_F16) with_group(std::integral_constant<int, CAKE_HIP_F16>());
    else with_group(std::integral_constant<int, CAKE_HIP_BF16>());
}

}  // namespace cake
