// Attention of drafted tokens in float32 on the matrix cores: 16 or 32 columns a workgroup, by how many the step has and what the
// registers hold beside a page of keys and one of values (heads of 112 and 128: 16).
#include "attention_tree_mfma.h"

namespace {
template <int HD>
int launch_hd(const TreeArgs& a, hipStream_t stream) {
  const long cols = (long)a.max_nodes * (a.n_heads / a.n_kv_heads);
  if constexpr (HD <= 96)
    if (cols > 16) return launch_tree<float, HD, 2>(a, stream);
  return launch_tree<float, HD, 1>(a, stream);
}
}  // namespace

int yalm_attn_tree_f32_mfma(const TreeArgs& a, hipStream_t stream) {
  switch (a.head_dim) {
    case 16: return launch_hd<16>(a, stream);
    case 32: return launch_hd<32>(a, stream);
    case 48: return launch_hd<48>(a, stream);
    case 64: return launch_hd<64>(a, stream);
    case 80: return launch_hd<80>(a, stream);
    case 96: return launch_hd<96>(a, stream);
    case 112: return launch_hd<112>(a, stream);
    case 128: return launch_hd<128>(a, stream);
  }
  return YALM_ERR_ARG;
}
