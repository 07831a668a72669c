// rope_freq.h -- angles per position of rotary embeddings, with the scalings
// for contexts longer than a model was trained on.  Host-only C++.
#pragma once

#include <stddef.h>

#include <string>
#include <vector>

#include "../../include/hale_moe.h"

namespace hale {

// Checks the configuration and computes the angle per position of each pair,
// in radians; false with a message where the configuration is refused.
bool rope_frequencies(const hale_rope_config& c, std::vector<double>* freq, std::string* err);

}  // namespace hale
