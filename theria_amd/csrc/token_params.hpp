// Parameter blocks and launchers of the token-side kernels (layer norm, embedding, linear cross entropy), shared by
// the kernel files and the C ABI layer (capi_tokens.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace theria {

int device_cu_count();
int fail(int code, const char* msg);            // records the thread's error message, returns code
int hip_status(hipError_t e, const char* what);  // THERIA_OK, or THERIA_ERR_HIP with the message

// A (rows, width) view with a contiguous last dimension.
struct Rows {
  const void* p;
  int64_t sr;  // elements from row to row
};
struct MutRows {
  void* p;
  int64_t sr;
};

// ------------------------------------------------------------------------------------------ layer norm
constexpr int kNormMaxWidth = 16384;

struct NormParams {
  int dtype, param_dtype;  // theria_dtype
  int64_t rows;
  int width;
  float eps;
  Rows x, dout, gdx;
  const void *weight, *bias;   // optional
  const void *gdw, *gdb;       // double backward: cotangents of dweight and dbias, optional
  MutRows y, dx, out_gx, out_gdout;  // the gradients are optional
  float *mean, *rstd;          // one of each row
  void *dw, *db, *out_gw;      // optional
  float* ws;                   // partial column sums, norm_ws_floats() of them
};
int64_t norm_ws_floats(const NormParams& p);
hipError_t launch_norm_fwd(const NormParams& p, hipStream_t st);
hipError_t launch_norm_bwd(const NormParams& p, hipStream_t st);
hipError_t launch_norm_bwd_bwd(const NormParams& p, hipStream_t st);

// ------------------------------------------------------------------------------------------ embedding
struct EmbedParams {
  int dtype;
  bool ids64;
  bool zero_padding;  // lookup: rows of the padding id are zeros (the gradient's own lookup)
  int64_t n, classes;
  int width;
  float scale;
  int64_t padding;  // -1: none
  const void* ids;
  Rows table;    // lookup
  MutRows out;   // lookup: n rows; gradient: `classes` rows
  Rows dout;     // gradient
  void* ws;
};
int64_t embed_ws_bytes(const EmbedParams& p);
hipError_t launch_embed_fwd(const EmbedParams& p, hipStream_t st);
hipError_t launch_embed_bwd(const EmbedParams& p, hipStream_t st);

// ------------------------------------------------------------------------------------------ linear cross entropy
enum CeReduction : int { kCeNone = 0, kCeMean = 1, kCeSum = 2 };

struct CeParams {
  int dtype;
  bool target64;
  int reduction;  // CeReduction
  int64_t n, classes, ignore;
  int width;
  Rows x, w;
  const void *target, *bias;  // bias optional
  float* loss;                // n (kCeNone) or one
  float* stats;               // 2 n: of the i-th kept row, the largest logit and the sum of exp(logit - largest); few
                              // classes (ce_head_takes): the number of kept rows in the first place
  const float* gout;          // backward: n (kCeNone) or one
  MutRows dx, dw;             // optional
  void* db;                   // optional
  void* ws;
};
int64_t ce_ws_bytes(const CeParams& p, bool backward);
hipError_t launch_ce_fwd(const CeParams& p, hipStream_t st);
hipError_t launch_ce_bwd(const CeParams& p, hipStream_t st);
// Few classes (linear_ce_head.hip).
bool ce_head_takes(const CeParams& p);
int64_t ce_head_ws_bytes(const CeParams& p, bool backward);
hipError_t launch_ce_head(const CeParams& p, bool backward, hipStream_t st);

}  // namespace theria
