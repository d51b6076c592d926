// token_gemm_bf16.hip -- token_gemm.h for bfloat16 operands.
#include "token_gemm.h"

int token_launch_bf16(int form, int tile, bool direct, const TokenArgs& a, hipStream_t s)
{
    switch (form)
    {
        case LVG_TOKEN_FORWARD:  return token_launch_form<bf16_t, bf16_t, ALONG, ALONG, false>(tile, direct, a, s);
        case LVG_TOKEN_GATED:    return token_launch_form<bf16_t, bf16_t, ALONG, ALONG, true>(tile, direct, a, s);
        case LVG_TOKEN_ROW_GRAD: return token_launch_form<bf16_t, bf16_t, DOWN, ALONG, false>(tile, direct, a, s);
        default:                 return token_launch_form<bf16_t, bf16_t, DOWN, DOWN, false>(tile, direct, a, s);
    }
}
