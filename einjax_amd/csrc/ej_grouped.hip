// Products grouped by expert: argument checks and the choice of kernel.
#include "ej_grouped.h"

#include "ej_grouped_launch.h"

namespace ej {
namespace {

bool aligned16(const void *p, int64_t a, int64_t b, int size) {
  return reinterpret_cast<size_t>(p) % 16 == 0 && a * size % 16 == 0 && b * size % 16 == 0;
}

// The kernels count slots in 32 bits, up to two blocks or stages past the last.
constexpr int64_t kMaxSlots = (int64_t{1} << 31) - 512;

int elem_size(int32_t dtype) { return dtype == EJ_F32 ? 4 : dtype == EJ_I8 ? 1 : 2; }

int check_desc(const ej_grouped_desc *d) {
  EJ_CHECK_ARG(d, "null descriptor");
  EJ_CHECK_ARG(d->dtype == EJ_F32 || d->dtype == EJ_BF16 || d->dtype == EJ_F16 ||
                   d->dtype == EJ_I8,
               "operands of dtype %d: expected EJ_F32, EJ_BF16, EJ_F16 or EJ_I8", d->dtype);
  EJ_CHECK_ARG(d->w_order == EJ_W_KN || d->w_order == EJ_W_NK, "w_order = %d", d->w_order);
  EJ_CHECK_ARG(d->n_groups >= 0 && d->k >= 0 && d->n >= 0 && d->n_slots >= 0 && d->n_rows >= 0,
               "negative size");
  const int64_t w_row = d->w_order == EJ_W_KN ? d->n : d->k;
  const int64_t w_rows = d->w_order == EJ_W_KN ? d->k : d->n;
  EJ_CHECK_ARG(d->x_stride >= d->k && d->out_stride >= d->n && d->w_stride >= w_row,
               "a row stride is below its row's length");
  EJ_CHECK_ARG(d->n_groups <= 1 || d->w_group >= w_rows * d->w_stride || w_rows * w_row == 0,
               "groups of w overlap: stride %lld for %lld rows of %lld", (long long)d->w_group,
               (long long)w_rows, (long long)d->w_stride);
  if (d->n_slots > kMaxSlots || d->n_rows >= (int64_t{1} << 31)) {
    set_error("%lld slots of %lld rows: at most %lld slots and fewer than 2^31 rows are supported",
              (long long)d->n_slots, (long long)d->n_rows, (long long)kMaxSlots);
    return EJ_E_UNSUPPORTED;
  }
  return EJ_OK;
}

// Whether rows and weights can be loaded as whole, aligned chunks, going by the
// descriptor (the workspace is sized without the operands' addresses).
bool whole_chunks(const ej_grouped_desc *d) {
  const int size = elem_size(d->dtype), chunk = 16 / size;
  return d->k % chunk == 0 && aligned16(nullptr, d->x_stride, 0, size) &&
         aligned16(nullptr, d->w_stride, d->w_group, size) &&
         (d->w_order == EJ_W_NK || d->n % chunk == 0);
}

// Parts of the contraction, for 64 x 64 tiles that leave CUs without work and
// have a long way to go.  A part is a pass over its sums (`sums` elements,
// written and read at 4 TB/s), and adding the parts is a launch (5 us); a stage
// takes a workgroup 0.4 us in 16 bits and 0.7 in fp32, and twice that through
// registers, where more workgroups to a CU are of use.  Measured (us) in one
// part and in the parts taken:
//   rows product     256 x 4096 x 4096 bf16              27   23 (2)
//                    512 x 4096 x 64 bf16                27   11 (8)
//                    1515 x 3392 x 135 fp32, 25 groups   77   50 (5)
//                    45 x 1539 x 294 fp32, 30 groups     72   31 (8)
//   weight gradient  8192 rows, 128 x 128 bf16           49   10 (16)
//                    4096 rows, 1024 x 1024 bf16         28   25 (2)
//                    26556 rows, 6 groups, 311 x 215 f16 272  68 (8)
// and with 512 tiles 29 and 39 in two parts.
int split_parts(double tiles, int64_t contraction, int elem, bool whole, double sums) {
  const int64_t stages = contraction / (128 / elem);
  // fp32 tiles on every CU are bound by their matrix instructions (258 x 3608 x
  // 2497 in 6 groups, 281 tiles: 66 us, 78 in two parts)
  if (tiles <= 0 || stages < 8 || (whole && elem == 4 && tiles > 192)) return 1;
  const int64_t want = static_cast<int64_t>((whole ? 576 : 1152) / tiles);
  const int64_t most = whole ? stages / 8 : stages / 4, cap = whole ? 32 : 8;
  const int64_t parts = want < most && want < cap ? want : most < cap ? most : cap;
  if (parts < 2) return 1;
  const double saved = stages * (1 - 1. / parts) * (elem == 4 ? 0.7 : 0.4) * (whole ? 1 : 2);
  return saved > 5 + parts * sums * 8 / 4e6 ? static_cast<int>(parts) : 1;
}

int rows_parts(const ej_grouped_desc *d) {
  if (d->dtype == EJ_I8 || d->n_groups == 0 || d->n_slots == 0) return 1;
  const int64_t groups = d->n_groups < d->n_slots ? d->n_groups : d->n_slots;
  const double rows = static_cast<double>(d->n_slots) / groups;
  const double tiles = (rows / 64 + 0.5) * groups * ceil_div(d->n, 64);
  const int elem = elem_size(d->dtype);
  const bool whole = whole_chunks(d);
  // the kernel for few rows splits k by itself
  if (whole && few_rows(rows, tiles, elem) && (rows <= 16 || tiles > 64)) return 1;
  return split_parts(tiles, d->k, elem, whole, static_cast<double>(d->n_slots) * d->n);
}
int dw_parts(const ej_grouped_desc *d) {
  if (d->n_groups == 0) return 1;
  const int size = elem_size(d->dtype), chunk = 16 / size;
  const bool whole = d->k % chunk == 0 && d->n % chunk == 0 &&
                     aligned16(nullptr, d->x_stride, d->out_stride, size);
  const double tiles = static_cast<double>(ceil_div(d->k, 64)) * ceil_div(d->n, 64) * d->n_groups;
  return split_parts(tiles, d->n_slots / d->n_groups, size, whole,
                     static_cast<double>(d->n_groups) * d->k * d->n);
}

int check_workspace(int parts, int64_t sums, void *workspace, size_t bytes, GroupedArgs *g) {
  g->splits = parts;
  if (parts == 1) return EJ_OK;
  EJ_CHECK_ARG(workspace && bytes >= sizeof(float) * parts * sums,
               "workspace of %zu bytes, expected %zu", bytes, sizeof(float) * parts * sums);
  g->partial = static_cast<float *>(workspace);
  return EJ_OK;
}

}  // namespace
}  // namespace ej

using namespace ej;

extern "C" int ej_grouped_gemm_workspace_size(const ej_grouped_desc *d, size_t *bytes) {
  EJ_TRY(check_desc(d));
  EJ_CHECK_ARG(bytes, "null bytes");
  const int parts = rows_parts(d);
  *bytes = parts > 1 ? sizeof(float) * parts * d->n_slots * d->n : 0;
  return EJ_OK;
}

extern "C" int ej_grouped_gemm_dw_workspace_size(const ej_grouped_desc *d, size_t *bytes) {
  EJ_TRY(check_desc(d));
  EJ_CHECK_ARG(bytes, "null bytes");
  const int parts = dw_parts(d);
  *bytes = parts > 1 ? sizeof(float) * parts * d->n_groups * d->k * d->n : 0;
  return EJ_OK;
}

extern "C" int ej_grouped_gemm(const ej_grouped_desc *d, const void *x, const int32_t *rows,
                               const int32_t *offsets, const void *w, const float *x_scale,
                               const float *w_scale, void *out, void *workspace,
                               size_t workspace_bytes, ej_stream_t stream) {
  EJ_TRY(check_desc(d));
  const bool i8 = d->dtype == EJ_I8;
  EJ_CHECK_ARG(d->out_dtype == EJ_F32 || d->out_dtype == d->dtype ||
                   (i8 && (d->out_dtype == EJ_BF16 || d->out_dtype == EJ_F16)),
               "result of dtype %d from operands of dtype %d", d->out_dtype, d->dtype);
  EJ_CHECK_ARG(d->out_dtype != EJ_I8, "8-bit results are not products");
  if (i8) {
    EJ_CHECK_ARG(d->w_order == EJ_W_NK, "8-bit weights are k-contiguous (EJ_W_NK)");
    // |sum| <= 128 * 128 * k
    EJ_CHECK_ARG(d->k < (1 << 17), "k = %d: the 32-bit sum of 8-bit products holds k < 131072",
                 d->k);
  }
  if (d->n_slots == 0 || d->n == 0) return EJ_OK;
  EJ_CHECK_ARG(out, "null result");
  EJ_CHECK_ARG(offsets || d->n_groups == 1, "null offsets of %d groups", d->n_groups);
  EJ_CHECK_ARG(rows || d->n_rows >= d->n_slots, "%lld rows for %lld slots without a row index",
               (long long)d->n_rows, (long long)d->n_slots);
  EJ_CHECK_ARG(d->n_groups == 0 || d->n_rows > 0, "%lld slots of no rows",
               (long long)d->n_slots);
  EJ_CHECK_ARG(d->k == 0 || d->n_groups == 0 || (x && w), "null operand");
  EJ_CHECK_ARG(!i8 || d->n_groups == 0 || (x_scale && w_scale), "null scale");

  const int size = elem_size(d->dtype);
  GroupedArgs g = {};
  g.a = static_cast<const char *>(x);
  g.b = static_cast<const char *>(w);
  g.c = out;
  g.a_rows = rows;
  g.offsets = offsets;
  g.a_scale = x_scale;
  g.b_scale = w_scale;
  g.lda = d->x_stride;
  g.ldb = d->w_stride;
  g.ldc = d->out_stride;
  g.b_group = d->w_group;
  g.n_a = d->n_rows;
  g.slots = d->n_slots;
  g.n_groups = d->n_groups;
  g.n = d->n;
  g.k = d->k;
  g.out = d->out_dtype;
  // 16-byte loads need whole, aligned chunks in every row
  const int chunk = 16 / size;
  const bool direct = d->k % chunk == 0 && aligned16(x, d->x_stride, 0, size) &&
                      aligned16(w, d->w_stride, d->w_group, size) &&
                      (d->w_order == EJ_W_NK || d->n % chunk == 0);
  EJ_TRY(check_workspace(rows_parts(d), d->n_slots * d->n, workspace, workspace_bytes, &g));
  const GroupedRows r{g, d->w_order == EJ_W_NK, direct};
  switch (d->dtype) {
    case EJ_BF16: return grouped_rows_bf16(r, as_stream(stream));
    case EJ_F16: return grouped_rows_f16(r, as_stream(stream));
    case EJ_I8: return grouped_rows_i8(r, as_stream(stream));
    default: return grouped_rows_f32(r, as_stream(stream));
  }
}

extern "C" int ej_grouped_gemm_dw(const ej_grouped_desc *d, const void *x, const int32_t *rows,
                                  const int32_t *offsets, const void *grad, void *grad_w,
                                  void *workspace, size_t workspace_bytes, ej_stream_t stream) {
  EJ_TRY(check_desc(d));
  EJ_CHECK_ARG(d->dtype != EJ_I8, "8-bit products have no gradient");
  EJ_CHECK_ARG(d->out_dtype == EJ_F32 || d->out_dtype == d->dtype,
               "gradient of dtype %d from operands of dtype %d", d->out_dtype, d->dtype);
  if (d->n_groups == 0 || d->k == 0 || d->n == 0) return EJ_OK;
  EJ_CHECK_ARG(grad_w, "null result");
  EJ_CHECK_ARG(offsets || d->n_groups == 1, "null offsets of %d groups", d->n_groups);
  EJ_CHECK_ARG(rows || d->n_rows >= d->n_slots, "%lld rows for %lld slots without a row index",
               (long long)d->n_rows, (long long)d->n_slots);
  EJ_CHECK_ARG(d->n_slots == 0 || (d->n_rows > 0 && x && grad), "null operand");
  const int size = elem_size(d->dtype), chunk = 16 / size;
  GroupedArgs g = {};
  g.offsets = offsets;
  g.c = grad_w;
  g.c_group = d->w_group;
  g.ldc = d->w_stride;
  g.slots = d->n_slots;
  g.n_groups = d->n_groups;
  g.out = d->out_dtype;
  // the rows of D are k for [k][n] weights and n for [n][k]
  const bool kn = d->w_order == EJ_W_KN;
  const char *xp = static_cast<const char *>(x), *gp = static_cast<const char *>(grad);
  g.a = kn ? xp : gp;
  g.a_rows = kn ? rows : nullptr;
  g.lda = kn ? d->x_stride : d->out_stride;
  g.n_a = kn ? d->n_rows : d->n_slots;
  g.m = kn ? d->k : d->n;
  g.b = kn ? gp : xp;
  g.b_rows = kn ? nullptr : rows;
  g.ldb = kn ? d->out_stride : d->x_stride;
  g.n_b = kn ? d->n_slots : d->n_rows;
  g.n = kn ? d->n : d->k;
  EJ_TRY(check_workspace(dw_parts(d), static_cast<int64_t>(d->n_groups) * d->k * d->n, workspace,
                         workspace_bytes, &g));
  const bool direct = d->k % chunk == 0 && d->n % chunk == 0 &&
                      aligned16(x, d->x_stride, 0, size) &&
                      aligned16(grad, d->out_stride, 0, size);
  switch (d->dtype) {
    case EJ_BF16: return grouped_wgrad_bf16(g, direct, as_stream(stream));
    case EJ_F16: return grouped_wgrad_f16(g, direct, as_stream(stream));
    default: return grouped_wgrad_f32(g, direct, as_stream(stream));
  }
}
