// fa_rotary_args.h -- the by-value kernel argument blocks of the rotary tables and
// of the rotation (host and device).
#pragma once
#include <stdint.h>

#include "fa_udiv.h"

namespace fa {

constexpr int kMaxAngles = 128;  // angles of a position: rotary_dim / 2

struct RotaryTableArgs {
    const void* positions;
    int wide;                    // positions in 64 bits
    int64_t n;
    int half;                    // angles of a position
    float factor;                // of cosines and sines
    void* cos;
    void* sin;
    double turns[kMaxAngles];    // quarter turns that angle i takes for a position
};

// x[0] is q, x[1] k (heads 0: there is none). A row is (batch, position) or, ragged,
// a token; strides are in elements.
struct RotaryArgs {
    const void* x[2];
    int64_t x_sb[2], x_si[2], x_sh[2];
    void* o[2];
    int64_t o_sb[2], o_si[2], o_sh[2];
    int heads0, heads;           // of q, of both
    int hd, rd;
    int in_place;                // what is not rotated stays
    float sign;                  // -1: the other way round
    const void* cos;
    const void* sin;
    int64_t c_stride, s_stride;  // rows of the tables
    int seqlen_ro;
    const void* positions;       // of every row, or null
    int wide;
    int64_t p_sb, p_si;
    const int* offsets;          // of a sequence's first row, or null
    int64_t offset;
    const int* cu;               // ragged: starts of the sequences, or null
    int B;
    int64_t rows, row0;          // row0: first of the launch
    uint32_t items;              // work items of the launch
    UDiv seqlen, per_row, units; // division by the rows of a sequence, the items of a row, the units of a head row
};

}  // namespace fa
