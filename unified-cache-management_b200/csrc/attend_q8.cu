// Attention over listed blocks of the quantised cache, 8 bits (kernel: attend.cuh).
#include "attend.cuh"

namespace ucmx {
namespace attend {
int32_t run_q8(const Params& p, int head_dim, int cols, const Maps* maps, Plan* plan, cudaStream_t st)
{
    return run_format<8>(p, head_dim, cols, maps, plan, st);
}
}  // namespace attend
}  // namespace ucmx
