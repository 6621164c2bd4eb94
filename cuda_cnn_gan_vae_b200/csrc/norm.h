// Argument checks shared by the layer-normalisation and checkpoint entry points.
#pragma once
#include <cstddef>

namespace b200 {

constexpr size_t kMaxRow = ((size_t)1 << 31) - 65536;   // values in a row, and rows: their numbers and a grid of rows beyond stay in 31 bits
int check_rows(int rows, size_t n);
int check_matrix(const void *p, int type, int rows, size_t n, size_t pitch, const char *name);
int check_ckpt8(const void *codes, const void *exponents);

}  // namespace b200
