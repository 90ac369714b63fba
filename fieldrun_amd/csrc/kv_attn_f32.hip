// kv_attn_f32.hip — paged attention over an f32 cache (kv_attn.h), gfx950.
#include "kv_attn.h"

namespace frq {
namespace kv {
hipError_t launch_decode_f32(const Args& a, const Launch& l) { return launch_decode<FRQ_DT_F32, false>(a, l); }
hipError_t launch_prompt_f32(const Args& a, const Launch& l) { return launch_prompt<FRQ_DT_F32, false>(a, l); }
}  // namespace kv
}  // namespace frq
