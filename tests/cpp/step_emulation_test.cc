// The embedding kernels (csrc/step_embedding.hip) compiled for the CPU and run
// under the sanitizers: exact-size buffers, so every access outside one is an
// error, and results against plain loops in 64 bits.
#include <stdint.h>
#include <stdio.h>
#include <stdlib.h>
#include <string.h>

#include <cmath>
#include <map>
#include <random>
#include <vector>

#include "step_abi.h"

namespace {

int g_cases = 0;
#define REQUIRE(x)                                                                                   \
  do {                                                                                               \
    if (!(x)) {                                                                                      \
      printf("FAILED %s:%d: %s (tokens %zu rows %zu width %zu stride %zu dtype %d ids %d kind %d)\n", \
             __FILE__, __LINE__, #x, c.tokens, c.rows, c.width, c.stride, c.dtype, c.id_type, c.kind); \
      exit(1);                                                                                       \
    }                                                                                                \
  } while (0)

struct Case {
  size_t tokens, rows, width, stride;
  int dtype, id_type, kind;
};

float half_to_float(uint16_t h) { _Float16 x; memcpy(&x, &h, 2); return static_cast<float>(x); }
float load(const char* p, int dtype) {
  if (dtype == STEP_F32) { float f; memcpy(&f, p, 4); return f; }
  uint16_t h;
  memcpy(&h, p, 2);
  if (dtype == STEP_F16) return half_to_float(h);
  const uint32_t u = static_cast<uint32_t>(h) << 16;
  float f;
  memcpy(&f, &u, 4);
  return f;
}
void store(char* p, int dtype, float f) {
  if (dtype == STEP_F32) { memcpy(p, &f, 4); return; }
  uint16_t h;
  if (dtype == STEP_F16) {
    const _Float16 x = static_cast<_Float16>(f);
    memcpy(&h, &x, 2);
  } else {
    uint32_t u;
    memcpy(&u, &f, 4);
    h = static_cast<uint16_t>((u + 0x7fff + ((u >> 16) & 1)) >> 16);
  }
  memcpy(p, &h, 2);
}
size_t size_of(int dtype) { return dtype == STEP_F32 ? 4 : 2; }
// half a unit in the last place of a value's type
double half_step(int dtype) { return dtype == STEP_F32 ? 0x1p-24 : dtype == STEP_F16 ? 0x1p-11 : 0x1p-8; }

struct Block {  // exact-size, 256-byte aligned
  char* p;
  explicit Block(size_t bytes) : p(static_cast<char*>(aligned_alloc(256, bytes ? (bytes + 255) / 256 * 256 : 256))) {}
  ~Block() { free(p); }
};

// kind 0: uniform ids, 1: one id for almost all tokens, 2: few ids, 3: a third outside the table, 4: all outside,
// 5: ascending
std::vector<int64_t> make_ids(const Case& c, std::mt19937& rng) {
  std::vector<int64_t> ids(c.tokens);
  for (size_t t = 0; t < c.tokens; t++) {
    const int64_t any = static_cast<int64_t>(rng() % (c.rows ? c.rows : 1));
    switch (c.kind) {
      case 1: ids[t] = rng() % 16 ? static_cast<int64_t>(c.rows / 2) : any; break;
      case 2: ids[t] = any % 3; break;
      case 3: ids[t] = rng() % 3 ? any : (rng() % 2 ? -1 - any : static_cast<int64_t>(c.rows) + any); break;
      case 4: ids[t] = t % 2 ? -1 : static_cast<int64_t>(c.rows); break;
      case 5: ids[t] = static_cast<int64_t>(t * c.rows / (c.tokens ? c.tokens : 1)); break;
      default: ids[t] = any;
    }
  }
  return ids;
}

void run(const Case& c, unsigned seed) {
  g_cases++;
  std::mt19937 rng(seed);
  const std::vector<int64_t> ids = make_ids(c, rng);
  const size_t id_size = c.id_type == STEP_I32 ? 4 : 8, size = size_of(c.dtype);
  std::vector<char> raw_ids(c.tokens * id_size);
  for (size_t t = 0; t < c.tokens; t++) {
    const int32_t narrow = static_cast<int32_t>(ids[t]);
    memcpy(&raw_ids[t * id_size], id_size == 4 ? static_cast<const void*>(&narrow) : &ids[t], id_size);
  }
  auto inside = [&](size_t t) { return ids[t] >= 0 && ids[t] < static_cast<int64_t>(c.rows); };
  auto fill = [&](std::vector<char>& v) {
    for (size_t k = 0; k + size <= v.size(); k += size) store(&v[k], c.dtype, static_cast<float>(static_cast<int>(rng() % 2001) - 1000) / 256);
  };
  const float scale = 1.25f;

  // lookup: the exact product, rounded once
  std::vector<char> table(c.rows && c.width ? ((c.rows - 1) * c.stride + c.width) * size : 0);
  fill(table);
  std::vector<char> out(c.tokens * c.width * size, 0x55);
  REQUIRE(step_embedding_lookup(raw_ids.data(), c.id_type, c.tokens, table.data(), c.dtype, c.rows, c.width, c.stride, scale,
                                out.data(), nullptr) == STEP_OK);
  for (size_t t = 0; t < c.tokens; t++)
    for (size_t d = 0; d < c.width; d++) {
      char want[4];
      store(want, c.dtype, inside(t) ? scale * load(&table[(ids[t] * c.stride + d) * size], c.dtype) : 0.f);
      REQUIRE(memcmp(want, &out[(t * c.width + d) * size], size) == 0);
    }

  // gradient
  std::vector<char> grad(c.tokens && c.width ? ((c.tokens - 1) * c.stride + c.width) * size : 0);
  fill(grad);
  std::map<int64_t, std::vector<double>> sums, sizes;
  for (size_t t = 0; t < c.tokens; t++) {
    if (!inside(t)) continue;
    auto& s = sums[ids[t]];
    auto& a = sizes[ids[t]];
    s.resize(c.width);
    a.resize(c.width);
    for (size_t d = 0; d < c.width; d++) {
      const double g = load(&grad[(t * c.stride + d) * size], c.dtype);
      s[d] += g;
      a[d] += std::fabs(g);
    }
  }
  // each of at most n additions in 32 bits, the product and the rounding to the type are off by half a step
  auto near = [&](const char* got, double sum, double abs_sum) {
    const double want = sum * scale, slack = (c.tokens + 2) * 0x1p-24 * abs_sum * scale;
    return std::fabs(load(got, c.dtype) - want) <= slack + (std::fabs(want) + slack) * half_step(c.dtype) + 1e-30;
  };
  std::vector<char> dense(c.rows * c.width * size, 0x55), again(c.rows * c.width * size, 0x66);
  for (auto* to : {&dense, &again}) {
    const size_t bytes = step_embedding_gradient_workspace(c.tokens, c.rows, c.width);
    Block ws(bytes);
    memset(ws.p, to == &dense ? 0x00 : 0x01, (bytes + 255) / 256 * 256);   // it needs no initialisation
    REQUIRE(step_embedding_gradient(raw_ids.data(), c.id_type, c.tokens, grad.data(), c.dtype, c.rows, c.width, c.stride,
                                    scale, to->data(), ws.p, bytes, nullptr) == STEP_OK);
  }
  REQUIRE(dense == again);
  for (size_t v = 0; v < c.rows; v++) {
    const auto at = sums.find(static_cast<int64_t>(v));
    for (size_t d = 0; d < c.width; d++) {
      const char* got = &dense[(v * c.width + d) * size];
      if (at == sums.end()) REQUIRE(load(got, c.dtype) == 0.f);
      else REQUIRE(near(got, at->second[d], sizes[static_cast<int64_t>(v)][d]));
    }
  }

  // sum of slices: ascending, the same sums, nothing behind the last row touched
  const size_t most = c.tokens < c.rows ? c.tokens : c.rows;
  std::vector<char> out_ids(most * id_size, 0x77), values(most * c.width * size, 0x77);
  int64_t count = -1;
  const size_t bytes = step_sum_slices_workspace(c.tokens, c.rows, c.width);
  Block ws(bytes);
  REQUIRE(step_sum_slices(raw_ids.data(), c.id_type, c.tokens, grad.data(), c.dtype, c.rows, c.width, c.stride, scale,
                          out_ids.data(), values.data(), &count, ws.p, bytes, nullptr) == STEP_OK);
  if (c.width) REQUIRE(count == static_cast<int64_t>(sums.size()));
  size_t u = 0;
  for (const auto& at : sums) {
    int64_t id = 0;
    if (id_size == 4) { int32_t narrow; memcpy(&narrow, &out_ids[u * 4], 4); id = narrow; }
    else memcpy(&id, &out_ids[u * 8], 8);
    REQUIRE(id == at.first);
    // the same bits as the dense gradient's row
    if (c.width) REQUIRE(memcmp(&values[u * c.width * size], &dense[at.first * c.width * size], c.width * size) == 0);
    u++;
  }
  for (size_t k = u * c.width * size; k < values.size(); k++) REQUIRE(values[k] == 0x77);
  for (size_t k = u * id_size; k < out_ids.size(); k++) REQUIRE(out_ids[k] == 0x77);
}

void refusals() {
  const Case c = {4, 8, 4, 4, STEP_F32, STEP_I64, 0};
  int64_t ids[4] = {0, 1, 2, 3}, count;
  float v[32] = {}, out[32];
  Block ws(4096);
  REQUIRE(step_embedding_lookup(ids, STEP_F32, 4, v, STEP_F32, 8, 4, 4, 1.f, out, nullptr) == STEP_ERR_DTYPE);
  REQUIRE(step_embedding_lookup(ids, STEP_I64, 4, v, STEP_I32, 8, 4, 4, 1.f, out, nullptr) == STEP_ERR_DTYPE);
  REQUIRE(step_embedding_lookup(nullptr, STEP_I64, 4, v, STEP_F32, 8, 4, 4, 1.f, out, nullptr) == STEP_ERR_ARGUMENT);
  REQUIRE(step_embedding_lookup(ids, STEP_I64, 4, nullptr, STEP_F32, 8, 4, 4, 1.f, out, nullptr) == STEP_ERR_ARGUMENT);
  REQUIRE(step_embedding_lookup(ids, STEP_I64, 4, v, STEP_F32, 8, 4, 3, 1.f, out, nullptr) == STEP_ERR_ARGUMENT);
  REQUIRE(step_embedding_lookup(ids, STEP_I64, 4, v, STEP_F32, 8, 4, 4, 1.f, nullptr, nullptr) == STEP_ERR_ARGUMENT);
  REQUIRE(step_embedding_lookup(ids, STEP_I64, size_t(1) << 31, v, STEP_F32, 8, 4, 4, 1.f, out, nullptr) == STEP_ERR_LIMIT);
  REQUIRE(step_embedding_lookup(ids, STEP_I64, 4, v, STEP_F32, size_t(1) << 31, 4, 4, 1.f, out, nullptr) == STEP_ERR_LIMIT);
  REQUIRE(step_embedding_lookup(ids, STEP_I64, 4, v, STEP_F32, 8, 67107841, 67107841, 1.f, out, nullptr) == STEP_ERR_LIMIT);
  const size_t need = step_embedding_gradient_workspace(4, 8, 4);
  REQUIRE(step_embedding_gradient(ids, STEP_I64, 4, v, STEP_F32, 8, 4, 4, 1.f, out, ws.p, need - 1, nullptr) == STEP_ERR_ARGUMENT);
  REQUIRE(step_embedding_gradient(ids, STEP_I64, 4, v, STEP_F32, 8, 4, 4, 1.f, out, nullptr, need, nullptr) == STEP_ERR_ARGUMENT);
  REQUIRE(step_embedding_gradient(ids, STEP_I64, 4, v, STEP_F32, 8, 4, 4, 1.f, out, ws.p + 64, need, nullptr) == STEP_ERR_ARGUMENT);
  REQUIRE(step_embedding_gradient(ids, STEP_I64, 4, v, STEP_F32, 8, 4, 4, 1.f, nullptr, ws.p, need, nullptr) == STEP_ERR_ARGUMENT);
  REQUIRE(step_sum_slices(ids, STEP_I64, 4, v, STEP_F32, 8, 4, 4, 1.f, ids, out, nullptr, ws.p, 4096, nullptr) == STEP_ERR_ARGUMENT);
  REQUIRE(step_sum_slices(ids, STEP_I64, 4, v, STEP_F32, 8, 4, 4, 1.f, nullptr, out, &count, ws.p, 4096, nullptr) == STEP_ERR_ARGUMENT);
  REQUIRE(step_embedding_gradient_workspace(size_t(1) << 31, 8, 4) == 0);
}

}  // namespace

int main(int argc, char** argv) {
  const bool brief = argc > 1 && !strcmp(argv[1], "brief");
  refusals();
  unsigned seed = 1;
  const int types[3] = {STEP_F32, STEP_BF16, STEP_F16};
  const size_t tokens[] = {0, 1, 2, 63, 64, 65, 127, 129, 300, 700, 1023, 1024, 1025, 1700, 1536, 1537};
  const size_t widths[] = {1, 7, 8, 33, 65};
  for (size_t k = 0; k < sizeof(tokens) / sizeof(tokens[0]); k++) {
    for (int kind = 0; kind < 6; kind++) {
      if (brief && (k + kind) % 4) continue;
      const size_t rows[] = {1, 5, 31, 32, 100, 1100};
      const size_t width = widths[(k + kind) % 5];
      run({tokens[k], rows[(k * 5 + kind) % 6], width, width + (k % 3) * 3, types[(k + kind) % 3], kind % 2 ? STEP_I32 : STEP_I64, kind}, seed++);
    }
  }
  run({130, 40, 2100, 2100, STEP_BF16, STEP_I64, 2}, seed++);   // a row wider than a workgroup
  run({200, 3, 300, 301, STEP_F32, STEP_I32, 1}, seed++);       // whole waves to a row, long runs
  for (int kind = 0; kind < 6; kind++) run({300, 40, 131, 135, types[kind % 3], STEP_I64, kind}, seed++);
  run({500, 12, 264, 264, STEP_BF16, STEP_I32, 0}, seed++);
  run({130, 2, 257, 260, STEP_BF16, STEP_I64, 0}, seed++);
  run({5, 0, 4, 4, STEP_F32, STEP_I64, 4}, seed++);             // an empty table
  run({5, 9, 0, 0, STEP_F32, STEP_I64, 0}, seed++);             // no columns
  printf("step emulation: ok (%d cases)\n", g_cases);
  return 0;
}
