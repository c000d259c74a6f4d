// The orthogonalisation's kernels (csrc/step_orthogonalize.hip) compiled for
// the CPU and run under the sanitizers: exact-size buffers, so every access
// outside one is an error, and results against plain loops in 64 bits.
#include <stdint.h>
#include <stdio.h>
#include <stdlib.h>
#include <string.h>

#include <algorithm>
#include <cmath>
#include <random>
#include <vector>

#include "step_abi.h"
#include "step_matrix_shim.h"

namespace step {
int hip_fail(hipError_t) { return STEP_ERR_HIP; }  // step_embedding.hip's
}  // namespace step

namespace {

int g_cases = 0;

struct Shape {
  size_t rows, cols, count;
};
struct Case {
  std::vector<Shape> shapes;
  int dtype, out_dtype, precise, steps;
  unsigned side;
  bool muon;
};

void fail(const Case& c, const char* what, double got, double bound) {
  printf("FAILED: %s: %g, at most %g (", what, got, bound);
  for (const Shape& s : c.shapes) printf("%zu of %zu x %zu, ", s.count, s.rows, s.cols);
  printf("dtype %d to %d, precise %d, steps %d, side %u, muon %d)\n", c.dtype, c.out_dtype, c.precise, c.steps, c.side, c.muon);
  exit(1);
}

size_t size_of(int dtype) { return dtype == STEP_F32 ? 4 : 2; }
double half_step(int dtype) { return dtype == STEP_F32 ? 0x1p-24 : dtype == STEP_F16 ? 0x1p-11 : 0x1p-8; }
float load(const void* at, size_t i, int dtype) {
  if (dtype == STEP_F32) return static_cast<const float*>(at)[i];
  const uint16_t h = static_cast<const uint16_t*>(at)[i];
  if (dtype == STEP_F16) {
    _Float16 x;
    memcpy(&x, &h, 2);
    return static_cast<float>(x);
  }
  const uint32_t u = static_cast<uint32_t>(h) << 16;
  float f;
  memcpy(&f, &u, 4);
  return f;
}
void store(void* at, size_t i, int dtype, float f) {
  if (dtype == STEP_F32) {
    static_cast<float*>(at)[i] = f;
    return;
  }
  uint16_t h;
  if (dtype == STEP_F16) {
    const _Float16 x = static_cast<_Float16>(f);
    memcpy(&h, &x, 2);
  } else {
    uint32_t u;
    memcpy(&u, &f, 4);
    h = static_cast<uint16_t>((u + 0x7fff + ((u >> 16) & 1)) >> 16);
  }
  static_cast<uint16_t*>(at)[i] = h;
}

// What the steps make of a matrix, by rows, in 64 bits.
std::vector<double> exact(std::vector<double> u, size_t rows, size_t cols, const std::vector<float>& abc, float eps) {
  const bool tall = rows > cols;
  const size_t m = std::min(rows, cols), n = std::max(rows, cols);
  double norm = 0;
  for (double x : u) norm += x * x;
  norm = std::sqrt(norm) + static_cast<double>(eps);
  std::vector<double> x(m * n);
  for (size_t i = 0; i < m; i++)
    for (size_t j = 0; j < n; j++) x[i * n + j] = u[tall ? j * cols + i : i * cols + j] / norm;
  std::vector<double> a(m * m), b(m * m), next(m * n);
  for (size_t step = 0; 3 * step < abc.size(); step++) {
    for (size_t i = 0; i < m; i++)
      for (size_t k = 0; k <= i; k++) {
        double sum = 0;
        for (size_t j = 0; j < n; j++) sum += x[i * n + j] * x[k * n + j];
        a[i * m + k] = a[k * m + i] = sum;
      }
    for (size_t i = 0; i < m; i++)
      for (size_t k = 0; k < m; k++) {
        double sum = 0;
        for (size_t j = 0; j < m; j++) sum += a[i * m + j] * a[j * m + k];
        b[i * m + k] = abc[3 * step + 1] * a[i * m + k] + abc[3 * step + 2] * sum + (i == k ? abc[3 * step] : 0.0);
      }
    std::fill(next.begin(), next.end(), 0.0);
    for (size_t i = 0; i < m; i++)
      for (size_t k = 0; k < m; k++)
        for (size_t j = 0; j < n; j++) next[i * n + j] += b[i * m + k] * x[k * n + j];
    x.swap(next);
  }
  for (size_t i = 0; i < m; i++)
    for (size_t j = 0; j < n; j++) u[tall ? j * cols + i : i * cols + j] = x[i * n + j];
  return u;
}

void run(const Case& c) {
  std::mt19937 rng(7 + g_cases);
  std::normal_distribution<float> normal;
  step_matrix_shim::g_side = c.side;
  const float momentum = 0.9f, keep = 0.75f, eps = 1e-7f;
  std::vector<float> abc;
  for (int k = 0; k < c.steps; k++) abc.insert(abc.end(), {3.4445f - 0.1f * k, -4.7750f, 2.0315f});
  std::vector<void*> grads, outs;
  std::vector<float*> buffers;
  std::vector<step_matrix> list;
  std::vector<std::vector<double>> before, updates, next_buffers;
  for (const Shape& s : c.shapes) {
    const size_t size = s.rows * s.cols * s.count;
    // exactly as large as they are
    void* grad = malloc(size * size_of(c.dtype) + (size ? 0 : 1));
    void* out = malloc(size * size_of(c.out_dtype) + (size ? 0 : 1));
    float* buffer = c.muon ? static_cast<float*>(malloc(size * 4 + (size ? 0 : 1))) : nullptr;
    before.emplace_back(size);
    updates.emplace_back(size);
    next_buffers.emplace_back(size);
    for (size_t i = 0; i < size; i++) {
      store(grad, i, c.dtype, 0.01f * normal(rng));
      store(out, i, c.out_dtype, normal(rng));
      const double g = load(grad, i, c.dtype);
      updates.back()[i] = g;
      before.back()[i] = load(out, i, c.out_dtype);
      if (c.muon) {
        buffer[i] = 0.01f * normal(rng);
        next_buffers.back()[i] = static_cast<double>(momentum) * buffer[i] + g;
        updates.back()[i] = g + static_cast<double>(momentum) * next_buffers.back()[i];
      }
    }
    grads.push_back(grad);
    outs.push_back(out);
    buffers.push_back(buffer);
    list.push_back({grad, buffer, out, s.rows, s.cols, s.count, 0.5f + list.size()});
  }
  const size_t bytes = step_orthogonalize_workspace(list.data(), list.size(), c.precise);
  void* workspace = bytes ? aligned_alloc(256, bytes) : nullptr;   // a multiple of 256, exactly
  if (bytes) memset(workspace, 0x7f, bytes);                       // NaN in every plane: what nobody wrote shows
  const int rc = c.muon ? step_muon(list.data(), list.size(), c.dtype, c.precise, c.steps, abc.data(), eps, momentum, 1, keep, workspace, bytes, nullptr)
                        : step_orthogonalize(list.data(), list.size(), c.dtype, c.out_dtype, c.precise, c.steps, abc.data(), eps, workspace, bytes, nullptr);
  if (rc != STEP_OK) fail(c, "status", rc, 0);
  for (size_t k = 0; k < list.size(); k++) {
    const Shape& s = c.shapes[k];
    const size_t one = s.rows * s.cols;
    const bool fine = c.precise || (std::min(s.rows, s.cols) <= 64 && std::max(s.rows, s.cols) <= 256);
    for (size_t j = 0; j < s.count && one; j++) {
      const auto first = updates[k].begin() + j * one;
      const std::vector<double> o = exact({first, first + one}, s.rows, s.cols, abc, eps);
      double off = 0, moved = 0, all = 0;
      for (size_t i = 0; i < one; i++) {
        const double step = c.muon ? list[k].rate * o[i] : o[i];
        const double want = c.muon ? keep * before[k][j * one + i] - step : step;
        const double d = load(outs[k], j * one + i, c.out_dtype) - want;
        off += d * d;
        moved += step * step;
        all += want * want;
        if (c.muon) {
          // one product and one sum in 32 bits
          const double m = next_buffers[k][j * one + i], e = std::fabs(buffers[k][j * one + i] - m);
          if (e > 0x1p-23 * (std::fabs(m) + 0.1)) fail(c, "momentum", e, 0x1p-23 * (std::fabs(m) + 0.1));
        }
      }
      // split operands: 1e-5. Single ones: what is documented, 0.3 % from eight rows on, 0.6 % below.
      const double bound = (fine ? 1e-5 : std::min(s.rows, s.cols) >= 8 ? 0.003 : 0.006) * std::sqrt(moved) + (half_step(c.out_dtype) + 0x1p-21) * std::sqrt(all);
      if (!(std::sqrt(off) <= bound)) fail(c, "result", std::sqrt(off), bound);
    }
  }
  for (size_t k = 0; k < list.size(); k++) {
    free(grads[k]);
    free(outs[k]);
    free(buffers[k]);
  }
  free(workspace);
  g_cases++;
}

}  // namespace

int main(int argc, char** argv) {
  const bool brief = argc > 1 && !strcmp(argv[1], "brief");
  const int F = STEP_F32, B = STEP_BF16, H = STEP_F16;
  // matrices of one workgroup: both widths, tall and wide, odd ends, more than one of them
  run({{{3, 5, 2}}, F, F, 1, 2, 0, false});
  run({{{64, 129, 1}, {30, 17, 3}, {1, 1, 1}}, B, B, 0, 2, 0, true});
  // products in every tile side, cut by the matrix's edge; an odd and an even number of stages
  run({{{70, 130, 1}}, F, F, 0, 3, 64, false});
  run({{{130, 70, 2}}, B, H, 0, 1, 64, false});
  run({{{65, 300, 1}}, F, F, 1, 2, 64, false});
  run({{{130, 200, 1}}, F, B, 0, 2, 128, false});
  if (!brief) {
    run({{{250, 64, 1}, {64, 256, 1}, {7, 9, 1}}, H, F, 1, 2, 0, false});
    run({{{1, 300, 1}, {300, 2, 1}, {64, 257, 1}}, F, F, 0, 3, 64, false});
    run({{{200, 140, 1}}, H, H, 1, 2, 128, false});
    run({{{140, 321, 1}, {70, 100, 2}, {20, 30, 1}, {0, 900, 1}, {100, 100, 0}}, B, B, 0, 2, 128, true});
    run({{{140, 190, 1}, {20, 30, 2}, {64, 500, 1}}, F, F, 1, 1, 128, true});
    run({{{200, 210, 1}}, F, F, 0, 2, 192, false});
    run({{{321, 200, 1}}, F, F, 0, 2, 256, true});
    // more batches, more shapes and more elements than a round holds
    run({{{5, 300, 1}, {6, 310, 1}, {7, 320, 1}, {320, 8, 1}}, F, F, 0, 1, 64, true});
    run({{{9, 300, 1}, {9, 400, 1}, {9, 450, 1}, {300, 9, 1}}, F, F, 1, 1, 64, false});
    run({{{65, 66, 4}}, F, F, 0, 1, 64, false});
    run({{{1, 2, 1}, {3, 200, 1}, {5, 5, 1}, {200, 2, 1}, {6, 6, 1}, {7, 7, 2}}, B, B, 0, 1, 0, true});
  }
  printf("step orthogonalize emulation: ok (%d cases)\n", g_cases);
  return 0;
}
