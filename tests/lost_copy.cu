// The norm and its gradient with one bulk copy that never starts: the wait for
// its row runs out.  Built by the test that loads it; nothing else differs from
// the library's own kernels.
#include "cmb_device.cuh"

namespace cmb {
namespace dev {

__device__ unsigned long long lost_row;  // its address; 0: none

__device__ __forceinline__ void bulk_load_but_lost(uint32_t dst, const void *src, uint32_t bytes,
                                                   uint32_t bar) {
  if (reinterpret_cast<unsigned long long>(src) != lost_row) bulk_load(dst, src, bytes, bar);
}

}  // namespace dev
}  // namespace cmb

#define bulk_load bulk_load_but_lost
#include "rmsnorm.cu"
#undef bulk_load

extern "C" int lose_row(unsigned long long address) {
  return cudaMemcpyToSymbol(cmb::dev::lost_row, &address, sizeof(address)) == cudaSuccess ? 0 : 1;
}
