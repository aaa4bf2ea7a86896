// The tiled products of the pair log probabilities of half precision values.
#include "tp_pairs_products.hh"

namespace tp {
template struct PairProducts<F16>;
}  // namespace tp
