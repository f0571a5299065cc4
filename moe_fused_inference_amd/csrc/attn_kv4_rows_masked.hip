// attn_kv4_rows_masked.hip -- the kernels of attn_kv4_rows.h with masks (windows, trees).
#include "attn_kv4_rows.h"

int mxa::attn_rows_masked(const Args& a, int q_dtype, const Plan& p, int D, bool exact, hipStream_t st) {
    return launch_rows<true>(a, q_dtype, p, D, exact, st);
}
