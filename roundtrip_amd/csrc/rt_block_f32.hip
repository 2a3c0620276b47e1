// rt_block_f32.hip — see rt_block_launch.hpp.
#include "rt_internal.hpp"
#define RT_BLOCK_DT RT_F32
#include "rt_block_launch.hpp"
