// Chunk kernels of the selective scan for bf16 activations (one file per type: they compile side by side).
#include "ssm_scan_chunk.h"

namespace mb {
namespace ssm {

int scan_chunks_bf16(const mb_selective_scan_args& a, const Split& sp, bool states, hipStream_t s) { return chunk_launch<bf16>(a, sp, states, s); }

}  // namespace ssm
}  // namespace mb
