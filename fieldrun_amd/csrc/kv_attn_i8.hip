// kv_attn_i8.hip — paged attention over an int8 cache (kv_attn.h), gfx950.
#include "kv_attn.h"

namespace frq {
namespace kv {
hipError_t launch_decode_i8(const Args& a, const Launch& l) { return launch_decode<FRQ_DT_ROWI8>(a, l); }
hipError_t launch_prompt_i8(const Args& a, const Launch& l) { return launch_prompt<FRQ_DT_ROWI8>(a, l); }
}  // namespace kv
}  // namespace frq
