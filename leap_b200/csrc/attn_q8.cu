// attn_q8.cu — attention over the 8-bit KV cache: which kernel takes a call.
#include "q8.cuh"

namespace leap {

int q8_attend(leap_ctx *c, int layer, const Q8Seqs &tab, const Q8Tree *tree, const float *q,
              const float *k, const float *v, float *out) {
    if (tab.tok0[tab.n_seq] == 0) return LEAP_OK;
    int most = 0;
    for (int i = 0; i < tab.n_seq; ++i)
        if (tab.tok0[i + 1] - tab.tok0[i] > most) most = tab.tok0[i + 1] - tab.tok0[i];
    if (most * c->group <= kQ8Rows) return q8_rows_attend(c, layer, tab, tree, q, k, v, out);
    return q8_tc_attend(c, layer, tab, tree, q, k, v, out);
}

}  // namespace leap
