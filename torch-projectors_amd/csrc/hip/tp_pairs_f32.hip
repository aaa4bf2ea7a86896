// The tiled products of the pair log probabilities of float32 values.
#include "tp_pairs_products.hh"

namespace tp {
template struct PairProducts<F32>;
}  // namespace tp
