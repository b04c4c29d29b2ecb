// Host harness for the plan of vbs_cu_attention_tree (test infrastructure, no
// GPU): reads, one line each,
//   head_dim kv_heads seqs group tokens window weights clusters step limit
// and prints, for ctx_limit = step, 2 step, .. limit, what tree_plan needs and
// what tree_bytes returns. `clusters` is how many CTAs of a kernel fit the GPU
// at once as clusters (0: none). tests/test_tree_plan.py compiles it; the
// library's tree.cu is part of it, its neighbours are stubs.
#include "tree.cu"

#include <cstdio>
#include <vector>

namespace vbs {
void note_launches(uint64_t) {}
void latch_error(const char *, ...) {}
bool cuda_ok(cudaError_t, const char *) { return false; }
DevState *backend_current() { return nullptr; }
bool kv_desc_ok(const vbs_cu_kv_t *) { return true; }
bool overlap(const void *, uint64_t, const void *, uint64_t) { return false; }
cudaError_t tree_tc_configure(int *) { return cudaErrorUnknown; }
cudaError_t tree_tc_launch(const TreeParams &, const CUtensorMap &, const CUtensorMap &, uint32_t, uint32_t, cudaStream_t) { return cudaErrorUnknown; }
cudaError_t tree_weights_configure() { return cudaErrorUnknown; }
cudaError_t tree_weights_launch(const TreeParams &, const CUtensorMap &, uint32_t, int, cudaStream_t) { return cudaErrorUnknown; }
}  // namespace vbs

int main() {
    unsigned hd, nkh, seqs, group, tokens, window, weights, clusters, step, limit;
    static float one;
    while (scanf("%u %u %u %u %u %u %u %u %u %u", &hd, &nkh, &seqs, &group, &tokens, &window, &weights, &clusters, &step, &limit) == 10) {
        for (auto &f : tree_fit)
            for (unsigned c = 2; c <= TREE_CLUSTER; ++c) f[c] = (int)(clusters / c);
        vbs_cu_kv_t kv = {};
        kv.n_kv_heads = nkh; kv.n_seqs = seqs; kv.head_dim = hd; kv.max_ctx = limit;
        vbs_cu_tree_t t = {};
        t.n_q_heads = nkh * group; t.n_tokens = tokens; t.window = window; t.weights_out = weights ? &one : nullptr;
        for (unsigned l = step; l <= limit; l += step) {
            t.ctx_limit = l;
            const TreePlan pl = tree_plan(&kv, &t, 148);
            printf("%zu:%zu:%u:%u:%d ", pl.bytes, tree_bytes(&kv, &t, 148), pl.tile_rows, pl.n_splits, (int)pl.joined);
        }
        printf("\n");
    }
    return 0;
}
