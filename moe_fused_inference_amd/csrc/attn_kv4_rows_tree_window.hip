// attn_kv4_rows_tree_window.hip -- the kernels of attn_kv4_rows.h with trees and a window.
#include "attn_kv4_rows.h"

int mxa::attn_rows_tree_window(const Args& a, int q_dtype, const Plan& p, int D, bool exact, hipStream_t st) {
    return launch_rows<kWindow | kTree>(a, q_dtype, p, D, exact, st);
}
