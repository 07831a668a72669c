// Runs the launchers of the 4-bit products (hale-token_amd/csrc/kernels_q4g.hip, host pass) over a HIP
// runtime that only notes launches: over many sizes and types every launch is within the device's
// limits, and a kernel's limit of LDS is the same in every call, so that calls of two
// contexts cannot lower it between another's setting and launch.  Exits 1 with a message where it
// fails.
#include <stdio.h>
#include <stdlib.h>

#include <map>
#include <vector>

#include "kernels.h"
#include "step_ops.h"

using namespace hale;

#define CHECK(cond)                                                    \
  do {                                                                 \
    if (!(cond)) {                                                     \
      fprintf(stderr, "line %d: %s does not hold\n", __LINE__, #cond); \
      exit(1);                                                         \
    }                                                                  \
  } while (0)

struct Launch {
  const void* kernel;
  dim3 grid, block;
  size_t lds;
};
static std::vector<Launch> launches;
static std::map<const void*, int> limits;

extern "C" {
extern const char no_device_code[1] = {0};
void** __hipRegisterFatBinary(const void*) { return nullptr; }
void __hipUnregisterFatBinary(void**) {}
void __hipRegisterFunction(void**, const void*, char*, const char*, unsigned, void*, void*, void*, void*, int*) {}
hipError_t __hipPopCallConfiguration(dim3*, dim3*, size_t*, hipStream_t*) { return hipSuccess; }
hipError_t hipFuncSetAttribute(const void* kernel, hipFuncAttribute a, int v) {
  CHECK(a == hipFuncAttributeMaxDynamicSharedMemorySize && v > 65536 && v <= 163840);
  CHECK(!limits.count(kernel) || limits[kernel] == v);
  limits[kernel] = v;
  return hipSuccess;
}
hipError_t hipLaunchKernel(const void* kernel, dim3 grid, dim3 block, void**, size_t lds, hipStream_t) {
  launches.push_back({kernel, grid, block, lds});
  return hipSuccess;
}
hipError_t hipExtLaunchKernel(const void*, dim3, dim3, void**, size_t, hipStream_t, hipEvent_t, hipEvent_t, int) { return hipSuccess; }
}

namespace hale {
ProfEvents& prof_events() {
  static ProfEvents e;
  return e;
}
}  // namespace hale

int main() {
  for (size_t rows : {1, 16, 40, 300, 1001, 4096, 6200, 16400, 24600, 151936})
    for (size_t cols : {32, 512, 2048, 4224, 14336})
      for (unsigned group : {32, 64, 128})
        for (size_t ntok : {1, 2, 7, 13, 16, 17, 48, 130, 1000, 70000, 1 << 20})
          for (int in : {Q4G_F32, Q4G_F16, Q4G_BF16, Q4G_I8})
            for (unsigned shift : {5, 6, 7, 31})
              for (bool bf16 : {false, true}) {
                if (cols % group || (in != Q4G_I8 && shift != 31) || (shift < 31 && cols % (1u << shift)) || ntok * rows > ((size_t)1 << 35)) continue;
                static uint8_t mem[64];
                Q4gArgs a{};
                a.g.data = mem, a.g.rows = rows, a.g.cols = cols, a.g.group = group, a.g.per = 128 / group;
                a.g.chunks = (unsigned)((cols + 127) / 128), a.g.bf16 = bf16;
                a.x = a.out = mem, a.x_scales = (const float*)mem, a.x_stride = cols;
                a.x_shift = shift, a.x_per = shift == 31 ? 1 : (unsigned)(cols >> shift);
                a.ntok = ntok, a.out_dtype = in == Q4G_F32 ? HALE_F32 : HALE_BF16, a.out_stride = rows;
                launches.clear();
                CHECK(launch_q4g((Q4gInput)in, a, nullptr) == hipSuccess && !launches.empty());
                for (const Launch& l : launches) {
                  CHECK(l.lds <= 163840 && (l.lds <= 65536 || (limits.count(l.kernel) && (size_t)limits[l.kernel] >= l.lds)));
                  CHECK((uint64_t)l.grid.x * l.block.x < 1ull << 32 && l.grid.y < 65536 && l.grid.z < 65536);
                  CHECK(l.grid.x && l.grid.y && l.grid.z && l.block.x <= 1024 && l.block.x % 64 == 0);
                  if (l.grid.y > 1) CHECK((size_t)l.grid.x * l.grid.y * l.grid.z <= q4g_part_tiles((rows + 15) / 16));
                }
              }
  CHECK(limits.size() > 10);
  return 0;
}
