// The kernel of ryft.paged_attention for many rows a sequence (k_paged_prompt.hip), called by k_paged_attention.hip.
#pragma once

#include "kernels.h"
#include "prompt_tiles.h"

namespace ryft {

void paged_prompt_plan(PagedAttnArgs& a, int64_t* ws_floats);
void launch_paged_prompt(const PagedAttnArgs& a, hipStream_t stream, hipEvent_t done);

}  // namespace ryft
