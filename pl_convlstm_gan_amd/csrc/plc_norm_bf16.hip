// Group norm kernels of one element type (see plc_norm_launch.h).
#define PLC_NORM_TYPE 1
#include "plc_norm_launch.h"

int plc_norm_launch_bf16(const NormArgs& a, const NormPlan& pl, bool backward, hipStream_t st) {
    return norm_type<plc_bf16>(a, pl, backward, st);
}
