// The tiled products of the pair log probabilities of bfloat16 values.
#include "tp_pairs_products.hh"

namespace tp {
template struct PairProducts<BF16>;
}  // namespace tp
