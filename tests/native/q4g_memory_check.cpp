// Checks the memory of 4-bit matrices (hale-token_amd/csrc/step_ops.hip) over a HIP runtime in host
// memory (kv_fake_hip.h), under AddressSanitizer and UndefinedBehaviorSanitizer: little more than
// their bytes, and all that a launch's divided rows can need.  Exits 1 with a message where it
// fails.
#include <malloc.h>

#include "kv_fake_hip.h"
#include "step_ops.h"

using namespace hale;

static Q4gGeom last;

namespace hale {
hipError_t launch_norm_q8(int, const NormQ8Args&, size_t, hipStream_t) { return hipSuccess; }
hipError_t launch_q4g_pack(const Q4gGeom& g, const uint8_t*, const uint16_t*, const uint8_t*, hipStream_t) {
  last = g;
  return hipSuccess;
}
hipError_t launch_q4g_unpack(const Q4gGeom&, uint8_t*, uint16_t*, uint8_t*, hipStream_t) { return hipSuccess; }
hipError_t launch_q4g(Q4gInput, const Q4gArgs&, hipStream_t) { return hipSuccess; }
hipError_t launch_logits(int, const LogitsArgs&, size_t, hipStream_t) { return hipSuccess; }
}  // namespace hale

static size_t held() {
  size_t n = 0;
  for (void* p : fake.device) n += malloc_usable_size(p);
  return n;
}

int main() {
  hale_ctx c;
  for (size_t rows : {1, 16, 100, 1000, 2048, 2064, 16000})
    for (bool with_zeros : {false, true}) {
      const size_t cols = 2048, groups = rows * (cols / 64);
      std::vector<uint8_t> codes(rows * cols / 2), zeros(groups);
      std::vector<uint16_t> scales(groups);
      hale_q4g* m = nullptr;
      CHECK(hale_q4g_upload(&c, rows, cols, 64, HALE_F16, codes.data(), scales.data(), with_zeros ? zeros.data() : nullptr, &m) == HALE_OK);
      const size_t tiles = (rows + 15) / 16, weights = tiles * last.tile_bytes;
      CHECK(weights <= (tiles * 16) * (cols / 2 + cols / 64 * (with_zeros ? 3 : 2)) + 128 * tiles);
      CHECK(held() <= weights + (rows <= 2048 ? 260 * 1024 : 0) + 64);
      // partial sums and counters of every launch lie within what was allocated, before the zeros that
      // a matrix without any reads
      const uint8_t* end = last.data + held() - 64;
      CHECK(with_zeros || last.zero_data == end);
      for (size_t slices = 1; slices <= 20; slices++)
        for (unsigned most : {1, 2, 5, 100}) {
          const size_t splits = q4g_splits(tiles, slices, most);
          CHECK(splits >= 1 && splits <= most);
          if (splits == 1) continue;
          CHECK((const uint8_t*)last.parts >= last.data + weights && (const uint8_t*)(last.parts + slices * splits * tiles * 256) <= (const uint8_t*)last.done);
          CHECK((const uint8_t*)(last.done + slices * tiles) <= end);
          for (size_t k = 0; k < slices * tiles; k++) CHECK(last.done[k] == 0);
        }
      hale_q4g_destroy(m);
      CHECK(fake.device.empty());
    }
  return 0;
}
