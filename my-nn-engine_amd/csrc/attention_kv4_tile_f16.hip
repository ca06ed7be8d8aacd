#include "attention_kv4_go.h"

namespace mynn {
template int kv4_tile_go<f16_t>(const Kv4Args &, int, int, const Kv4TilePlan &, hipStream_t);
}
