// Which products over narrow rows linear_stream.h has kernels for, and their launch shapes.
#include "linear_stream.h"

bool ngs_stream_forward_takes(long long rows, int k, int n, int dtype)
{
    if (rows <= NGS_FEW_ROWS || k < 1 || n < 1) return false;
    // As soon as there are more than a few rows: one launch, where the tiles cut the reduction and need a second
    // (1000 rows 250 -> 200 bfloat16 11 us, 18 us in tiles; there and back, 128 -> 128, three launches instead of six).
    // (16 steps of floats hold too many registers beside the results: 200000 x 200 -> 256 230 us in tiles, 356 us here)
    return steps_of(k, dtype) <= 8 && n <= 2 * 8 * 64 / (int)ngs_decoder_size(dtype);
}

bool ngs_stream_backward_takes(long long rows, int k, int n, int dtype)
{
    if (rows < 1 || k < 1 || n < 1) return false;
    const int size = (int)ngs_decoder_size(dtype), ks = steps_of(k, dtype), ns = steps_of(n, dtype);
    return ks <= 4 * size && ns <= 4 * size && ks * ns <= stream_most(size);  // a width of 256
}

long long ngs_stream_backward_blocks(long long rows, int k, int n, int dtype)
{
    const int size = (int)ngs_decoder_size(dtype), ks = steps_of(k, dtype), ns = steps_of(n, dtype);
    const int tm = stream_waves(ks, ns, size) * 16;
    const long long tiles = (rows + tm - 1) / tm, most = NGS_CUS * stream_per_cu(ks, ns, size);
    return tiles < most ? tiles : most;
}

