// Which products over narrow rows linear_stream.h has kernels for, and their launch shapes.
#include "linear_stream.h"

bool ngs_stream_forward_takes(long long rows, int k, int n, int dtype)
{
    if (rows < NGS_STREAM_ROWS || k < 16 / (int)ngs_decoder_size(dtype) || n < 1) return false;
    const int steps = steps_of(k, dtype);
    return steps <= 8 && n <= 2 * 8 * 64 / (int)ngs_decoder_size(dtype);
}

static int stream_waves(int ks, int ns) { return ks * ns > 32 ? 4 : 8; }
static size_t stream_backward_lds(int ks, int ns, int dtype)
{
    const int tn = ns * 64 / (int)ngs_decoder_size(dtype), tm = stream_waves(ks, ns) * 16;
    return (size_t)tn * ks * 64 + (size_t)tm * (ks + ns) * 64 + tn * 4;
}

// Rows of x and of dz of at most four steps, or eight steps of floats
bool ngs_stream_backward_takes(long long rows, int k, int n, int dtype)
{
    if (rows < NGS_STREAM_ROWS || k < 16 / (int)ngs_decoder_size(dtype) || n < 1) return false;
    const int most = dtype == NGS_FLOAT32 ? 8 : 4;
    return steps_of(k, dtype) <= most && steps_of(n, dtype) <= most;
}

// A row's kernel is instantiated for 1, 2, 4 (and 8) steps each of x and dz
long long ngs_stream_backward_blocks(long long rows, int k, int n, int dtype)
{
    const int ks = steps_of(k, dtype), ns = steps_of(n, dtype), tm = stream_waves(ks, ns) * 16;
    const long long tiles = (rows + tm - 1) / tm, per_cu = (long long)(160 * 1024 / stream_backward_lds(ks, ns, dtype));
    const long long most = NGS_CUS * (per_cu < 1 ? 1 : per_cu < 4 ? per_cu : 4);
    return tiles < most ? tiles : most;
}

