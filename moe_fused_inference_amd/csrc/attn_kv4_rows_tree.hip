// attn_kv4_rows_tree.hip -- the kernels of attn_kv4_rows.h with trees.
#include "attn_kv4_rows.h"

int mxa::attn_rows_tree(const Args& a, int q_dtype, const Plan& p, int D, bool exact, hipStream_t st) {
    return launch_rows<kTree>(a, q_dtype, p, D, exact, st);
}
