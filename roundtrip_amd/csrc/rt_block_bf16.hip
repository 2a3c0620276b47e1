// rt_block_bf16.hip — see rt_block_launch.hpp.
#include "rt_internal.hpp"
#define RT_BLOCK_DT RT_BF16
#include "rt_block_launch.hpp"
