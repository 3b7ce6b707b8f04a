// The kernels of linear_stream.h for one element type (a translation unit each: they take a while to compile).
#include "linear_stream.h"

NGS_STREAM_INSTANCE(float)
