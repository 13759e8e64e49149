// cw_tree_tc.cu -- the tcgen05 kernel of cw_tree_attention takes no shape yet.
#include "cw_tree.cuh"
namespace cw {
bool tree_tc_takes(const cw_tree_attn_args&, const void*, const void*, const void*) { return false; }
int tree_tc_rows(const TreeArgs&) { return 128; }
int tree_tc_grid(cw_ctx*, const TreeArgs&) { return 1; }
int tree_tc_launch(cw_ctx*, const TreeArgs&, uint32_t, int) { return CW_ERR_UNSUPPORTED; }
}
