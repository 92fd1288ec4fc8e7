// dorado_amd/csrc/ops_attention.h — what the host half (ops_attention.hip) hands to the kernels (ops_attention_kernels.hip, compiled
// once per head size).
#pragma once
#include "ops.h"

// n / d for n < 2^31 by a multiplication
struct AttDiv {
    unsigned m, s;
    void set(unsigned d) {
        s = 0;
        while ((1ull << s) < d) ++s;
        m = d == 1 ? 0 : (unsigned)((1ull << (31 + s)) / d + 1);
    }
    __device__ __forceinline__ unsigned div(unsigned n) const { return m == 0 ? n : __umulhi(n, m) >> (s - 1); }
};

enum { ATT_NO_CAP, ATT_NEAR, ATT_FAR };     // forms of the cap, see AttScore

struct AttArgs {
    mibc_attention_args a;
    AttDiv by_pairs, by_splits, by_tiles, by_kv, by_group;
    int back, ahead;  // the window's limits, -1: none
    int group;        // query heads per key head
    int rows;         // q_tokens * group: row r = (token r / group, head r % group) of a (batch, key head) pair
    int pairs;        // batch * kv_heads
    int tiles;        // row tiles per pair
    int splits;       // parts the keys of a tile are split into, joined by the second launch if > 1
    unsigned groups;  // workgroups: pairs * tiles * splits
    int order;        // workgroup -> (pair, tile, split): 0 pairs innermost, 1 tiles innermost (one pair stays on one XCD)
    int twin;         // pairs 2 i and 2 i + 1, whose keys share cache lines, run on one XCD at the same time (pairs % 16 == 0)
    float scale2;     // scale * log2(e)
    int cap;          // its form
    float cap_in, cap_out;   // ATT_NEAR: 2 scale / cap log2(e), cap log2(e); ATT_FAR: scale / cap, cap / scale
    float *part_o;    // [pairs * rows][splits][D] f32
    float *part_l;    // [pairs * rows][splits] log2 of the sum
};

// tokens: the kernel for at most 16 rows per pair, else tiles of 128 rows
#define MIBC_ATT_DECLARE(D) int mibc_att_launch_##D(hipStream_t s, const AttArgs &p, bool tokens);
MIBC_ATT_DECLARE(32)
MIBC_ATT_DECLARE(64)
MIBC_ATT_DECLARE(96)
MIBC_ATT_DECLARE(128)
