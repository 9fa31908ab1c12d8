// Chunk kernels of the selective scan for f32 activations (one file per type: they compile side by side).
#include "ssm_scan_chunk.h"

namespace mb {
namespace ssm {

int scan_chunks_f32(const mb_selective_scan_args& a, const Split& sp, bool states, hipStream_t s) { return chunk_launch<float>(a, sp, states, s); }

}  // namespace ssm
}  // namespace mb
