// attn_kv4_rows_window.hip -- the kernels of attn_kv4_rows.h with a window.
#include "attn_kv4_rows.h"

int mxa::attn_rows_window(const Args& a, int q_dtype, const Plan& p, int D, bool exact, hipStream_t st) {
    return launch_rows<kWindow>(a, q_dtype, p, D, exact, st);
}
