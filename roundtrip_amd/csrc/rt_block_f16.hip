// rt_block_f16.hip — see rt_block_launch.hpp.
#include "rt_internal.hpp"
#define RT_BLOCK_DT RT_F16
#include "rt_block_launch.hpp"
