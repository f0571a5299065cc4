// attn_kv4_window.hip -- the kernels of attn_kv4_few.h with a window.
#include "attn_kv4_few.h"

int mxa::attn_few_window(const Args& a, int q_dtype, const Plan& p, int D, bool much, hipStream_t st) {
    return launch_few<kWindow>(a, q_dtype, p, D, much, st);
}
