// rope_freq.cpp -- see rope_freq.h.
#include "rope_freq.h"

#include <cmath>

namespace hale {

bool rope_frequencies(const hale_rope_config& c, std::vector<double>* freq, std::string* err) {
  auto no = [&](const char* why) {
    *err = why;
    return false;
  };
  const size_t r = c.rotary_dim;
  if (c.layout != HALE_ROPE_HALF && c.layout != HALE_ROPE_INTERLEAVED) return no("unknown layout");
  if (c.head_dim == 0 || c.head_dim > 1024) return no("head_dim outside 1..1024");
  if (r == 0 || r % 2 || r > c.head_dim) return no("rotary_dim must be even, from 2 to head_dim");
  if (!(c.base > 1.0) || !std::isfinite(c.base)) return no("base must be a finite number above 1");
  const float factor = (float)c.attention_factor;  // as the kernels take it
  if (!(factor > 0.0f) || !std::isfinite(factor)) return no("attention_factor must be positive, and a finite f32 number");
  if (c.scaling < HALE_ROPE_NONE || c.scaling > HALE_ROPE_PARTS) return no("unknown scaling");
  if (c.scaling != HALE_ROPE_NONE && (!(c.factor >= 1.0) || !std::isfinite(c.factor)))
    return no("factor must be a finite number from 1 on");
  if (c.scaling == HALE_ROPE_NTK && r == 2) return no("ntk scaling needs a rotary_dim above 2");
  if (c.scaling == HALE_ROPE_PARTS) {
    if (!(c.original_len > 0.0) || !std::isfinite(c.original_len)) return no("original_len must be positive");
    if (!std::isfinite(c.low) || !std::isfinite(c.high) || c.low < 0.0 || c.high <= c.low)
      return no("low and high must be 0 <= low < high");
  }
  const double n = (double)r;
  const double base = c.scaling == HALE_ROPE_NTK ? c.base * std::pow(c.factor, n / (n - 2.0)) : c.base;
  if (!std::isfinite(base)) return no("base times its scaling is not finite");
  freq->resize(r / 2);
  for (size_t i = 0; i < r / 2; i++) {
    double f = std::pow(base, -2.0 * (double)i / n);
    if (c.scaling == HALE_ROPE_LINEAR) {
      f /= c.factor;
    } else if (c.scaling == HALE_ROPE_PARTS) {
      // whole turns of the pair within the original length: pairs of fewer than
      // `low` are interpolated, of more than `high` kept, between them mixed
      const double turns = c.original_len * f / (2.0 * M_PI);
      double keep = (turns - c.low) / (c.high - c.low);
      keep = keep < 0.0 ? 0.0 : keep > 1.0 ? 1.0 : keep;
      f = f * keep + f / c.factor * (1.0 - keep);
    }
    (*freq)[i] = f;
  }
  return true;
}

}  // namespace hale
