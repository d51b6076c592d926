// token_gemm_8bit.hip -- token_gemm.h for e4m3 operands (forward products only; results in bfloat16 or float16).
#include "token_gemm.h"

int token_launch_8bit(int form, int tile, bool direct, int out_dtype, const TokenArgs& a, hipStream_t s)
{
    if (out_dtype == LVG_BF16)
        return form == LVG_TOKEN_GATED ? token_launch_form<e4m3_t, bf16_t, ALONG, ALONG, true>(tile, direct, a, s)
                                       : token_launch_form<e4m3_t, bf16_t, ALONG, ALONG, false>(tile, direct, a, s);
    return form == LVG_TOKEN_GATED ? token_launch_form<e4m3_t, f16_t, ALONG, ALONG, true>(tile, direct, a, s)
                                   : token_launch_form<e4m3_t, f16_t, ALONG, ALONG, false>(tile, direct, a, s);
}
