// token_stream.h -- forward products of at most 32 token rows (token_stream.hip), as token_finish.hip calls them.
#pragma once
#include "token_act.h"

struct e4m3_t { uint8_t bits; };

struct StreamArgs
{
    const void* w;             // [cols] (gated: [2 cols]) rows of `bytes` bytes
    const void* x;             // [rows] of them
    int64_t     ldw, ldx;      // bytes
    int64_t     bytes;
    int64_t     rows, cols;
    int         spans, spansPerSplit;
    float*      part;          // as in TokenArgs
    int64_t     ldpart;
    Finish      fin;
};

constexpr int64_t kStreamRows = 32, kStreamCols = (int64_t)1 << 26;       // (16 columns a workgroup of 512 threads; wider results go through the tiles)
int token_stream_splits(int64_t rows, int64_t cols, int64_t bytes, bool gated);
int token_stream_launch(const StreamArgs& a, int dtype, int out_dtype, bool gated, int splits, hipStream_t s);
