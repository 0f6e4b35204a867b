// Attention over the 8-bit cache (attention_q8.cuh) for widths padded to 128.
#include "attention_q8.cuh"

namespace cbis {
template int q8_run<128>(const Q8Args&, const Q8Plan&, bool, int, cudaStream_t);
}
