// kv_attn_ex_f16.hip — paged attention over an f16 cache with sinks or trees (kv_attn.h), gfx950.
#include "kv_attn.h"

namespace frq {
namespace kv {
hipError_t launch_decode_ex_f16(const Args& a, const Launch& l) { return launch_decode<FRQ_DT_F16, true>(a, l); }
hipError_t launch_prompt_ex_f16(const Args& a, const Launch& l) { return launch_prompt<FRQ_DT_F16, true>(a, l); }
}  // namespace kv
}  // namespace frq
