// Runs the host side of the norms, 4-bit products and logit rules
// (hale-token_amd/csrc/step_ops.hip) over a HIP runtime in host memory
// (kv_fake_hip.h), under AddressSanitizer and UndefinedBehaviorSanitizer.  The
// argument names the check; exits 1 with a message where it fails.
#include "kv_fake_hip.h"
#include "step_ops.h"

using namespace hale;

static int norms, packs, unpacks, products, rules;
static NormQ8Args last_norm;
static Q4gArgs last_q4g;
static LogitsArgs last_logits;

namespace hale {
hipError_t launch_norm_q8(int, const NormQ8Args& a, size_t, hipStream_t) {
  norms++;
  last_norm = a;
  return hipSuccess;
}
hipError_t launch_q4g_pack(const Q4gGeom& g, const uint8_t* codes, const uint16_t* scales, const uint8_t* zeros, hipStream_t) {
  packs++;
  // what the kernel reads and writes is there
  volatile uint8_t sum = 0;
  for (size_t i = 0; i < g.rows * (g.cols / 2); i++) sum = sum + codes[i];
  for (size_t i = 0; i < g.rows * (g.cols / g.group); i++) sum = sum + (uint8_t)scales[i] + (zeros ? zeros[i] : 0);
  memset(g.data, sum, (g.rows + Q4G_ROWS - 1) / Q4G_ROWS * g.tile_bytes);
  CHECK(g.scales_at == g.chunks * 1024 && g.tile_bytes % 128 == 0 && g.tile_bytes >= g.scales_at + g.chunks * g.per * (g.zeros ? 48 : 32));
  return hipSuccess;
}
hipError_t launch_q4g_unpack(const Q4gGeom& g, uint8_t* codes, uint16_t* scales, uint8_t* zeros, hipStream_t) {
  unpacks++;
  memset(codes, 0x12, g.rows * (g.cols / 2));
  memset(scales, 0x34, g.rows * (g.cols / g.group) * 2);
  memset(zeros, 5, g.rows * (g.cols / g.group));
  return hipSuccess;
}
hipError_t launch_q4g(Q4gInput, const Q4gArgs& a, hipStream_t) {
  products++;
  last_q4g = a;
  return hipSuccess;
}
hipError_t launch_logits(int, const LogitsArgs& a, size_t, hipStream_t) {
  rules++;
  last_logits = a;
  return hipSuccess;
}
}  // namespace hale

namespace {

alignas(16) char mem[1 << 16];

void norm_arguments() {
  hale_ctx c;
  float* f = (float*)mem;
  struct Call {
    int dtype = HALE_F32;
    size_t rows = 2, n = 64;
    const void* x = mem;
    size_t xs = 64;
    const void* delta = nullptr;
    size_t ds = 64;
    const float* w = (float*)mem;
    float eps = 1e-6f;
    size_t block = 32;
    void* sum = nullptr;
    size_t ss = 64;
    void* y = nullptr;
    size_t ys = 64;
    int8_t* q = (int8_t*)mem + 8192;
    float* scales = (float*)mem + 4096;
  };
  auto run = [&](const Call& a) {
    return hale_rms_norm_q8_device(&c, a.dtype, a.rows, a.n, a.x, a.xs, a.delta, a.ds, a.w, a.eps, a.block, a.sum, a.ss,
                                   a.y, a.ys, a.q, a.scales);
  };
  CHECK(run({}) == HALE_OK && norms == 1 && last_norm.vec && last_norm.block == 32);
  Call a;
  a.block = 64;  // as long as the row: still a block of lanes
  CHECK(run(a) == HALE_OK && last_norm.block == 64);
  a.n = a.xs = a.block = 96;
  CHECK(run(a) == HALE_OK && last_norm.block == 0);
  a = Call(), a.sum = mem;  // in place
  CHECK(run(a) == HALE_OK);
  a.ss = 65;
  CHECK(run(a) == HALE_EINVAL);
  a.rows = 1;
  CHECK(run(a) == HALE_OK && !last_norm.vec);
  a = Call(), a.x = mem + 4;
  CHECK(run(a) == HALE_OK && !last_norm.vec);
  a = Call(), a.q++;
  CHECK(run(a) == HALE_OK && !last_norm.vec);
  const int before = norms;
  auto refused = [&](const Call& b) { CHECK(run(b) == HALE_EINVAL && norms == before && !c.err.empty()); };
  a = Call(), a.dtype = HALE_Q8_0, refused(a);
  a = Call(), a.n = 0, refused(a);
  a = Call(), a.n = 65, refused(a);
  a = Call(), a.n = a.xs = NORM_Q8_MAX + 32, refused(a);
  for (size_t block : {0, 16, 48, 128}) a = Call(), a.block = block, refused(a);
  a = Call(), a.n = a.xs = 96, a.block = 64, refused(a);
  a = Call(), a.xs = 63, refused(a);
  a = Call(), a.delta = f, a.ds = 63, refused(a);
  a = Call(), a.sum = mem + 512, a.ss = 1, refused(a);
  a = Call(), a.y = mem + 512, a.ys = 1, refused(a);
  a = Call(), a.sum = a.y = mem + 512, refused(a);
  a = Call(), a.delta = mem + 512, a.y = mem + 512, a.ys = 80, refused(a);
  a = Call(), a.x = nullptr, refused(a);
  a = Call(), a.w = nullptr, refused(a);
  a = Call(), a.q = nullptr, refused(a);
  a = Call(), a.scales = nullptr, refused(a);
  a = Call(), a.x = mem + 2, refused(a);
  a = Call(), a.scales = (float*)(mem + 1), refused(a);
  for (int bits : {22, 31, 32}) a = Call(), a.rows = (size_t)1 << bits, refused(a);
  for (float eps : {-1.0f, __builtin_nanf(""), __builtin_inff()}) a = Call(), a.eps = eps, refused(a);
  a = Call(), a.rows = 0, a.x = nullptr;
  CHECK(run(a) == HALE_OK && norms == before);
  CHECK(hale_rms_norm_q8_device(nullptr, HALE_F32, 1, 32, mem, 32, nullptr, 0, f, 0, 32, nullptr, 0, nullptr, 0, (int8_t*)mem, f) == HALE_EINVAL);
}

void matrices() {
  hale_ctx c;
  hale_q4g* m = nullptr;
  std::vector<uint8_t> codes(33 * 48), zeros(33 * 3, 15);
  std::vector<uint16_t> scales(33 * 3);
  auto up = [&](size_t rows = 33, size_t cols = 96, size_t group = 32, int type = HALE_F16) {
    return hale_q4g_upload(&c, rows, cols, group, type, codes.data(), scales.data(), zeros.data(), &m);
  };
  CHECK(up() == HALE_OK && packs == 1 && fake.device.size() == 1);
  size_t rows, cols, group;
  int type, has;
  CHECK(hale_q4g_shape(m, &rows, &cols, &group, &type, &has) == HALE_OK && rows == 33 && cols == 96 && group == 32 && type == HALE_F16 && has);
  CHECK(hale_q4g_download(m, codes.data(), scales.data(), zeros.data()) == HALE_OK && unpacks == 1 && zeros[98] == 5 && codes.back() == 0x12);
  CHECK(hale_q4g_download(m, codes.data(), scales.data(), nullptr) == HALE_OK);
  // products
  auto f = [&](int dtype, size_t n, const void* x, size_t xs, void* o, size_t os) { return hale_q4g_matmul_device(m, dtype, n, x, xs, o, os); };
  CHECK(f(HALE_F32, 2, mem, 96, mem + 4096, 33) == HALE_OK && products == 1 && !last_q4g.out_vec && last_q4g.ntok == 2);
  CHECK(f(HALE_F32, 2, mem, 97, mem + 4096, 36) == HALE_OK && last_q4g.out_vec);
  CHECK(f(HALE_BF16, 2, mem, 104, mem + 4098, 40) == HALE_OK && !last_q4g.out_vec);
  auto q = [&](size_t block, const void* x, const void* s, size_t os) {
    return hale_q4g_matmul_q8_device(m, 2, block, (const int8_t*)x, (const float*)s, HALE_BF16, mem + 4096, os);
  };
  CHECK(q(32, mem, mem, 33) == HALE_OK && q(96, mem, mem, 33) == HALE_OK && last_q4g.x_shift == 31 && last_q4g.x_per == 1);
  const int before = products;
  CHECK(f(HALE_Q8_0, 2, mem, 96, mem, 33) == HALE_EINVAL && f(HALE_F32, 2, nullptr, 96, mem, 33) == HALE_EINVAL);
  CHECK(f(HALE_F32, 2, mem, 95, mem, 33) == HALE_EINVAL && f(HALE_F32, 2, mem, 96, mem, 32) == HALE_EINVAL);
  CHECK(f(HALE_F32, 2, mem + 2, 96, mem, 33) == HALE_EINVAL && f(HALE_F32, (1 << 20) + 1, mem, 96, mem, 33) == HALE_EINVAL);
  CHECK(q(0, mem, mem, 33) == HALE_EINVAL && q(64, mem, mem, 33) == HALE_EINVAL && q(48, mem, mem, 33) == HALE_EINVAL);
  CHECK(q(32, mem + 4, mem, 33) == HALE_EINVAL && q(32, mem, nullptr, 33) == HALE_EINVAL && q(32, mem, mem + 2, 33) == HALE_EINVAL);
  CHECK(f(HALE_F32, 0, nullptr, 96, nullptr, 33) == HALE_OK && products == before);
  CHECK(f(HALE_F32, 1 << 20, mem, 96, mem, 33) == HALE_OK && products == before + 1);
  fake.capturing = true;  // what allocates is refused inside a capture, what computes is recorded
  hale_q4g* other = nullptr;
  CHECK(hale_q4g_upload(&c, 33, 96, 32, HALE_F16, codes.data(), scales.data(), nullptr, &other) == HALE_EINVAL && !other);
  CHECK(hale_q4g_download(m, codes.data(), scales.data(), nullptr) == HALE_EINVAL);
  CHECK(f(HALE_F32, 2, mem, 96, mem, 33) == HALE_OK);
  fake.capturing = false;
  hale_q4g_destroy(m);
  CHECK(fake.device.empty());
  // refusals and failures leave nothing behind
  CHECK(up(0) == HALE_EINVAL && up(33, 0) == HALE_EINVAL && up(33, 80) == HALE_EINVAL && up(33, 96, 48) == HALE_EINVAL && up(33, 96, 64) == HALE_EINVAL);
  CHECK(up(33, 96, 32, HALE_F32) == HALE_EINVAL && up(((size_t)1 << 27) + 1) == HALE_EINVAL && !m);
  zeros[98] = 16;
  CHECK(up() == HALE_EINVAL && !m);
  zeros[98] = 0;
  for (int k = 0; k < 3; k++) {
    fake.allocs_until_failure = k;
    CHECK(up() == HALE_ENOMEM && !m && fake.device.empty());
    fake.allocs_until_failure = -1;
  }
  CHECK(up() == HALE_OK);
  fake.allocs_until_failure = 0;
  CHECK(hale_q4g_download(m, codes.data(), scales.data(), zeros.data()) == HALE_ENOMEM);
  fake.allocs_until_failure = -1;
  hale_q4g_destroy(m);
  hale_q4g_destroy(nullptr);
  CHECK(hale_q4g_matmul_device(nullptr, 0, 1, mem, 96, mem, 33) == HALE_EINVAL);
  CHECK(hale_q4g_matmul_q8_device(nullptr, 1, 32, (int8_t*)mem, (float*)mem, 0, mem, 33) == HALE_EINVAL);
  CHECK(hale_q4g_shape(nullptr, nullptr, nullptr, nullptr, nullptr, nullptr) == HALE_EINVAL);
}

void logit_arguments() {
  hale_ctx c;
  auto run = [&](const hale_logits_rules& r, size_t rows = 2, size_t vocab = 64, const void* x = mem, size_t xs = 64, void* o = mem + 4096,
                 size_t os = 64, int dtype = HALE_F32) { return hale_logits_device(&c, dtype, rows, vocab, x, xs, &r, o, os); };
  CHECK(run({}) == HALE_OK && rules == 1 && last_logits.vec);
  CHECK(run({}, 2, 64, mem, 64, mem) == HALE_OK && run({}, 1, 64, mem, 64, mem, 70) == HALE_OK);
  const int before = rules;
  CHECK(run({}, 2, 64, mem, 64, mem, 65) == HALE_EINVAL && run({}, 2, 64, nullptr) == HALE_EINVAL && run({}, 2, 64, mem, 63) == HALE_EINVAL);
  CHECK(run({}, 2, 64, mem, 64, mem, 64, HALE_Q4_0) == HALE_EINVAL && run({}, 2, (1 << 26) + 1, mem, 1 << 27, mem, 1 << 27) == HALE_EINVAL);
  CHECK(run({}, 2, 64, mem + 2) == HALE_EINVAL && run({}, (size_t)1 << 31) == HALE_EINVAL);
  hale_logits_rules r{};
  r.tokens = (int32_t*)mem;
  CHECK(run(r) == HALE_EINVAL);
  r.token_start = (int64_t*)(mem + 4);
  CHECK(run(r) == HALE_EINVAL);
  r = {};
  r.bias_tokens = (int32_t*)mem, r.bias = (float*)mem;
  CHECK(run(r) == HALE_EINVAL);
  r = {};
  r.mask = (uint32_t*)mem, r.mask_rows = 2, r.mask_stride = 1;
  CHECK(run(r) == HALE_EINVAL);
  r.mask_stride = 2, r.mask_rows = 1;
  CHECK(run(r) == HALE_EINVAL);
  r.mask_row = (int32_t*)(mem + 2);
  CHECK(run(r) == HALE_EINVAL);
  r = {}, r.ntokens = (size_t)1 << 31;
  CHECK(run(r) == HALE_EINVAL);
  CHECK(hale_logits_device(&c, HALE_F32, 1, 64, mem, 64, nullptr, mem, 64) == HALE_EINVAL);
  CHECK(hale_logits_device(nullptr, HALE_F32, 1, 64, mem, 64, &r, mem, 64) == HALE_EINVAL);
  CHECK(run({}, 0, 64, nullptr) == HALE_OK && run({}, 2, 0, nullptr) == HALE_OK && rules == before);
}

}  // namespace

int main(int argc, char** argv) {
  const std::string what = argc > 1 ? argv[1] : "";
  if (what == "norm_arguments") norm_arguments();
  else if (what == "matrices") matrices();
  else if (what == "logit_arguments") logit_arguments();
  else return 2;
  return 0;
}
