// Prints the rotary frequencies of the configuration given as arguments
// (layout scaling head_dim rotary_dim base factor original_len low high
// attention_factor), one per line, or "refused: <why>".
#include <stdio.h>
#include <stdlib.h>

#include "rope_freq.h"

int main(int argc, char** argv) {
  if (argc != 11) return 2;
  hale_rope_config c{};
  c.layout = atoi(argv[1]);
  c.scaling = atoi(argv[2]);
  c.head_dim = strtoul(argv[3], nullptr, 10);
  c.rotary_dim = strtoul(argv[4], nullptr, 10);
  c.base = strtod(argv[5], nullptr);
  c.factor = strtod(argv[6], nullptr);
  c.original_len = strtod(argv[7], nullptr);
  c.low = strtod(argv[8], nullptr);
  c.high = strtod(argv[9], nullptr);
  c.attention_factor = strtod(argv[10], nullptr);
  std::vector<double> f;
  std::string err;
  if (!hale::rope_frequencies(c, &f, &err)) {
    printf("refused: %s\n", err.c_str());
    return 0;
  }
  for (double v : f) printf("%.17g\n", v);
  return 0;
}
