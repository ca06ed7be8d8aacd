#include "attention_kv4_go.h"

namespace mynn {
template int kv4_stream_go<f16_t>(const Kv4Args &, int, int, int, int, hipStream_t);
}
