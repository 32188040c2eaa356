// Attention from the rows of one stream to another stream's: softmax(q k^T scale) v over the keys that a sample has
// (key_len) and does not mask (key_mask). q, k, v and out are strided (elements; the head's values are contiguous), key
// heads may be shared by H / Hkv query heads.
#pragma once

#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <cstdint>

namespace mkb {

struct HeadStrides {
    long row, head, sample;
};

struct CrossArgs {
    const __nv_bfloat16* q;
    const __nv_bfloat16* k;
    const __nv_bfloat16* v;
    __nv_bfloat16* out;
    HeadStrides sq, sk, sv, so;
    int B, H, Hkv, Lq, Lk, d;
    const int* key_len;       // [B] or null: Lk
    const uint8_t* key_mask;  // [B][Lk] rows mask_stride apart, 0: not seen; or null
    long mask_stride;
    float scale_log2;  // softmax scale * log2(e)
    uint32_t* status;
};
cudaError_t cross_attention(const CrossArgs& a, const char** err, cudaStream_t st);

}  // namespace mkb
