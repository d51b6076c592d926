// token_gemm_f32.hip -- token_gemm.h for float32 operands.
#include "token_gemm.h"

int token_launch_f32(int form, int tile, bool direct, const TokenArgs& a, hipStream_t s)
{
    switch (form)
    {
        case LVG_TOKEN_FORWARD:  return token_launch_form<float, float, ALONG, ALONG, false>(tile, direct, a, s);
        case LVG_TOKEN_GATED:    return token_launch_form<float, float, ALONG, ALONG, true>(tile, direct, a, s);
        case LVG_TOKEN_ROW_GRAD: return token_launch_form<float, float, DOWN, ALONG, false>(tile, direct, a, s);
        default:                 return token_launch_form<float, float, DOWN, DOWN, false>(tile, direct, a, s);
    }
}
