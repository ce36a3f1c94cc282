#include "paged_attention.cuh"

namespace bm {
namespace paged {

bool tc_takes(int, int, int, bm_dtype_t) { return false; }
size_t tc_workspace_bytes(int64_t, int64_t, int, int, int, int, int) { return 0; }
int launch_tc(const TreeArgs&, cudaStream_t, const char*) { return BM_OK; }

}  // namespace paged
}  // namespace bm
