// token_gemm_f16.hip -- token_gemm.h for float16 operands.
#include "token_gemm.h"

int token_launch_f16(int form, int tile, bool direct, const TokenArgs& a, hipStream_t s)
{
    switch (form)
    {
        case LVG_TOKEN_FORWARD:  return token_launch_form<f16_t, f16_t, ALONG, ALONG, false>(tile, direct, a, s);
        case LVG_TOKEN_GATED:    return token_launch_form<f16_t, f16_t, ALONG, ALONG, true>(tile, direct, a, s);
        case LVG_TOKEN_ROW_GRAD: return token_launch_form<f16_t, f16_t, DOWN, ALONG, false>(tile, direct, a, s);
        default:                 return token_launch_form<f16_t, f16_t, DOWN, DOWN, false>(tile, direct, a, s);
    }
}
