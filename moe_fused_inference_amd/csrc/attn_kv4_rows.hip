// attn_kv4_rows.hip -- the kernels of attn_kv4_rows.h without masks.
#include "attn_kv4_rows.h"

int mxa::attn_rows(const Args& a, int q_dtype, const Plan& p, int D, bool exact, hipStream_t st) {
    return launch_rows<0>(a, q_dtype, p, D, exact, st);
}
