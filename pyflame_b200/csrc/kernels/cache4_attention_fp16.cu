// cache4_attention_fp16.cu — the attention kernels over the 4-bit cache for one
// type of queries: three files, so that they compile side by side.
#define PFB_CACHE4_KERNELS
#include "cache4_attention.cuh"

namespace pfb {
namespace cache4 {

template int wave_of<__half>(int, int64_t, bool, bool);
template void launch_of<__half>(Args&, int, int64_t, bool, bool, int, cudaStream_t);

}  // namespace cache4
}  // namespace pfb
