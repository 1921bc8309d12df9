// (host_wave: see hip_runtime.h beside this)
#pragma once
#include "hip_runtime.h"
