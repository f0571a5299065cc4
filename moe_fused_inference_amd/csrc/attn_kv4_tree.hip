// attn_kv4_tree.hip -- the kernels of attn_kv4_few.h with trees.
#include "attn_kv4_few.h"

int mxa::attn_few_tree(const Args& a, int q_dtype, const Plan& p, int D, bool much, hipStream_t st) {
    return launch_few<kTree>(a, q_dtype, p, D, much, st);
}
