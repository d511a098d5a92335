// The sequences of a step, on the device: whose token a row is, its position, and the page that a position lies in.
#pragma once

#include "layer_common.h"

namespace cmoe {

// First new token and their number, of sequence b. Numbers that the caller got wrong never lead outside [0, tokens].
__device__ __forceinline__ void step_tokens(const StepView& s, int b, int& first, int& count) {
    if (!s.offsets) {
        first = b * s.uniform;
        count = s.uniform;
        return;
    }
    const int lo = s.offsets[b], hi = s.offsets[b + 1];
    first = lo < 0 ? 0 : lo > s.tokens ? s.tokens : lo;
    const int end = hi < first ? first : hi > s.tokens ? s.tokens : hi;
    count = end - first;
}

// The sequence that token t belongs to, s.seqs where it is behind the last one; asked by whole waves, the same t in all lanes.
__device__ __forceinline__ int step_sequence(const StepView& s, int t) {
    if (!s.offsets) return t / s.uniform;
    int before = 0;  // sequences whose tokens end at or before t
    for (int b0 = 0; b0 < s.seqs; b0 += 64) {
        const int b = b0 + (threadIdx.x & 63);
        const bool ended = b < s.seqs && s.offsets[b + 1] <= t;
        before += __popcll(__ballot(ended));
    }
    return __builtin_amdgcn_readfirstlane(before);
}

// The page of block `blk` of sequence b, -1 where the table has none or names one outside the pool.
__device__ __forceinline__ int step_page(const StepView& s, int b, int blk) {
    if (blk < 0 || blk >= s.blocks) return -1;
    const int page = s.table[b * s.table_stride + blk];
    return (unsigned)page < (unsigned)s.pages ? page : -1;
}

// One copy instruction of a wave, 16 bytes per lane, from a uniform base and a lane's own offset into 1 KB of LDS; waits and
// ordering are the caller's, as for dma16 (moe_tile.h).
__device__ __forceinline__ void dma16_at(const void* base, uint32_t offset, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %2\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(offset), "s"(base), "s"(lds) : "memory", "m0");
}

}  // namespace cmoe
