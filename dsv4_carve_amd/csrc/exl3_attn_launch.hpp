// How an attention call is divided, and the launches of each head size (exl3_attn_inst.hip).
#pragma once

#include <atomic>

#include "exl3_attn.hpp"

namespace exl3 {

struct AttnPlan {
    int rows;                    // of a tile: 16, 32, 64 or 128
    unsigned shares;             // workgroups of a launch that share the work, or 0: a workgroup a tile
    unsigned tiles;              // tiles at most, for a workgroup a tile
    int least;                   // units that a workgroup has at least
    int most;                    // workgroups that have units at most: whatever bounds the launch, the sums are divided alike
    unsigned join_rows;          // workgroups that join the rows of a tile
};

int launch_attention_64(const AttnArgs& A, const AttnPlan& P, bool bf16, hipStream_t s);
int launch_attention_128(const AttnArgs& A, const AttnPlan& P, bool bf16, hipStream_t s);
int launch_attention_192(const AttnArgs& A, const AttnPlan& P, bool bf16, hipStream_t s);
int launch_attention_256(const AttnArgs& A, const AttnPlan& P, bool bf16, hipStream_t s);

}  // namespace exl3
