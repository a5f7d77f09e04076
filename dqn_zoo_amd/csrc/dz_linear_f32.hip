// The dense-layer operator's kernels for float32 (a unit per type: they compile side by side).
#include "dz_linear_launch.h"

const DzLinearLaunch* dz_linear_launch_f32() { return linear_launches<float>(); }
