"""The integration guide's recipe of a step over a paged cache, compiled as it stands and run against
stand-ins of the entry points that check how the calls fit together."""
import os
import re
import subprocess

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

HARNESS = r"""
#include <cstdio>
#include <cstdlib>
#include "bm_layer_ops.h"

static const void* rotated = nullptr;
static int64_t rotated_stride = 0;
static int calls = 0;
#define NEED(x) if (!(x)) { std::printf("%s\n", #x); std::exit(1); }

extern "C" int bm_paged_kv_append(void* q_out, const void* q, const void*, const void*, const int32_t*, const int32_t*,
                                  const int32_t*, const bm_paged_kv_t* cache, const void*, int32_t, int32_t, int32_t,
                                  int64_t rows, int32_t num_q_heads, int64_t q_stride, int64_t, int64_t,
                                  int64_t q_out_stride, bm_dtype_t, int32_t*, void*) {
  ++calls;
  rotated = q_out;
  rotated_stride = q_out_stride;
  NEED(rows == 7 && q_out != nullptr && q_stride >= num_q_heads * cache->head_dim);
  return BM_OK;
}
extern "C" int bm_paged_tree_attention(void* out, const void* q, const bm_paged_kv_t* cache, const int32_t*, const int32_t*,
                                       const int32_t*, const uint64_t*, int32_t, int64_t total_q, int64_t batch,
                                       int32_t num_q_heads, int32_t, int32_t, float, void*, size_t, bm_dtype_t, int32_t*,
                                       void*) {
  ++calls;
  NEED(q == rotated);  // what the append rotated
  NEED(rotated_stride == num_q_heads * cache->head_dim);  // read as dense rows
  NEED(total_q == 7 && batch == 3 && out != nullptr && out != q);
  return BM_OK;
}
extern "C" int bm_sample(int32_t*, const void*, const float*, const float*, const int32_t*, const float*, const float*,
                         int64_t rows, int64_t vocab, int64_t row_stride, bm_dtype_t, int32_t*, void*) {
  ++calls;
  NEED(rows == 7 && row_stride >= vocab);
  return BM_OK;
}

// what the recipe takes as given: a server's own names
static char memory[64];
static void* k_pages[2] = {memory, memory};
static void* v_pages[2] = {memory + 16, memory + 16};
static int32_t ints[4], *page_table = ints, *positions = ints, *slots = ints, *seq_ids = ints, *ctx_lens = ints,
               *q_starts = ints, *top_k = ints, *tokens = ints, *d_status = ints;
static float floats[1], *uniforms = floats, *temperature = floats, *top_p = floats, *min_p = floats;
static uint64_t words[1], *tree_mask = words;
static void *q = memory + 24, *k = memory + 32, *v = memory + 40, *q_rot = memory + 48, *attn_out = memory + 56,
            *logits = memory, *rope_table = memory, *workspace = memory, *stream = nullptr;
static int l = 1, num_pages = 5, page_size = 16, max_pages = 2, n_seqs = 3, n_heads = 8, n_kv_heads = 2, head_dim = 64,
           max_pos = 100, R = 7, mask_words = 1, max_ctx = 20, max_tree = 4, vocab = 1000;
static int64_t q_stride = 12 * 64, k_stride = 12 * 64, v_stride = 12 * 64;  // slices of a fused projection
static size_t workspace_bytes = 64;

int main() {
RECIPE
  NEED(calls == 3);
  return 0;
}
"""


def test_the_recipe_of_a_paged_step(tmp_path):
    with open(os.path.join(REPO, "INTEGRATION.md")) as f:
        blocks = [b for b in re.findall(r"```cpp\n(.*?)```", f.read(), re.S) if "bm_paged_kv_append(" in b]
    assert len(blocks) == 1
    src, exe = tmp_path / "recipe.cpp", tmp_path / "recipe"
    src.write_text(HARNESS.replace("RECIPE", blocks[0]))
    built = subprocess.run(["g++", "-std=c++17", "-w", "-I", os.path.join(REPO, "include"), "-o", str(exe), str(src)],
                           capture_output=True, text=True)
    assert built.returncode == 0, built.stderr
    ran = subprocess.run([str(exe)], capture_output=True, text=True)
    assert ran.returncode == 0, ran.stdout
