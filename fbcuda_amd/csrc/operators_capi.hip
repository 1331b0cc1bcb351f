// C ABI of the operators around convolution and linear layers: argument validation and dispatch.
#include "operators.h"

#include <cmath>

using namespace fbfft_amd;

namespace {

constexpr long long kMost = 1ll << 40;  // elements of one array
constexpr long long kMostGroup = (1ll << 31) - (1 << 16);  // values of a group of group norm

bool okArray(const fbfft_array* a, int dim) {
  if (!a || a->dim != dim || a->type < FBFFT_FLOAT32 || a->type > FBFFT_BFLOAT16) return false;
  long long total = 1;
  for (int d = 0; d < dim; ++d) {
    if (a->size[d] < 0 || a->size[d] > kMost || a->stride[d] > kMost || a->stride[d] < -kMost) return false;
    total = total > kMost / (a->size[d] > 0 ? a->size[d] : 1) ? kMost + 1 : total * a->size[d];
  }
  if (total > kMost) return false;
  return total == 0 || (a->data && aligned(a->data, a->type == FBFFT_FLOAT32 ? 4 : 2));
}

bool sameShape(const fbfft_array* a, const fbfft_array* b) {
  if (a->dim != b->dim || a->type != b->type) return false;
  for (int d = 0; d < a->dim; ++d)
    if (a->size[d] != b->size[d]) return false;
  return true;
}

// a vector of n parameters, or none
bool okLine(const fbfft_array* a, long long n) { return !a || (okArray(a, 1) && a->size[0] == n); }
Line lineOf(const fbfft_array* a) { return a ? Line{a->data, (long)a->stride[0], a->type} : Line{}; }

bool okMatrix(const fbfft_array* a, long long rows, long long cols, int type) {
  return okArray(a, 2) && a->size[0] == rows && a->size[1] == cols && a->type == type;
}
Matrix matrixOf(const fbfft_array* a) { return a ? Matrix{a->data, (long)a->stride[0], (long)a->stride[1]} : Matrix{}; }

Image imageOf(const fbfft_array* a) {
  return a ? Image{a->data, (long)a->stride[0], (long)a->stride[1], (long)a->stride[2], (long)a->stride[3]} : Image{};
}

bool okActivation(int a) { return a >= FBFFT_ACTIVATION_NONE && a <= FBFFT_ACTIVATION_GELU; }

bool okWorkspace(const void* space, size_t bytes, size_t need) {
  return need == 0 || (space && aligned(space, 256) && bytes >= need);
}

bool okStatistics(const fbfft_array* a, const fbfft_array* input, long long groups) {
  return okArray(a, 2) && a->type == FBFFT_FLOAT32 && a->size[0] == input->size[0] && a->size[1] == groups;
}

// The shapes that both passes of group norm share; 0 or an error.
int checkNorm(const fbfft_array* input, const fbfft_array* weight, const fbfft_array* bias, long long groups, int activation) {
  if (!okArray(input, 4) || !okActivation(activation)) return FBFFT_UNSUPPORTED_DIMENSION;
  const long long C = input->size[1];
  if (groups < 1 || C % groups != 0) return FBFFT_UNSUPPORTED_SIZE;
  if (!okLine(weight, C) || !okLine(bias, C)) return FBFFT_UNSUPPORTED_DIMENSION;
  // (workgroups count images times channels, and lanes the values of a group in 31 bits.  A lane's place runs past a
  // group's end by less than 2^16: pieces rounded up to words add 2^14, words on their way 14336, rows of lanes 3584)
  if (input->size[0] * C > 0x7fffffff || C / groups * input->size[2] * input->size[3] > kMostGroup) return FBFFT_UNSUPPORTED_SIZE;
  return FBFFT_SUCCESS;
}

NormProblem normOf(const fbfft_array* input, const fbfft_array* weight, const fbfft_array* bias, const fbfft_array* mean,
                   const fbfft_array* rstd, long long groups, int activation, void* workspace) {
  NormProblem p{};
  p.x = imageOf(input);
  p.weight = lineOf(weight), p.bias = lineOf(bias);
  if (mean) p.mean = static_cast<float*>(mean->data), p.meanB = mean->stride[0], p.meanG = mean->stride[1];
  if (rstd) p.rstd = static_cast<float*>(rstd->data), p.rstdB = rstd->stride[0], p.rstdG = rstd->stride[1];
  p.B = input->size[0], p.C = input->size[1], p.G = groups, p.H = input->size[2], p.W = input->size[3];
  p.type = input->type, p.activation = activation, p.workspace = workspace;
  return p;
}

}  // namespace

extern "C" size_t fbfft_group_norm_workspace(int pass, long long batch, long long channels, long long pixels, long long groups) {
  if (pass < 0 || pass > 1 || batch <= 0 || channels <= 0 || pixels <= 0 || groups <= 0 || channels % groups != 0) return 0;
  if (batch > kMost / channels || batch * channels > 0x7fffffff || pixels > 0x7fffffff) return 0;
  return normWorkspaceBytes(pass, batch, channels, pixels, groups);
}

extern "C" int fbfft_group_norm_fprop(const fbfft_array* input, const fbfft_array* weight, const fbfft_array* bias,
                                      const fbfft_array* output, const fbfft_array* mean, const fbfft_array* rstd,
                                      long long groups, float eps, int activation, void* workspace, size_t workspaceBytes,
                                      fbfft_stream_t stream) {
  const int rc = checkNorm(input, weight, bias, groups, activation);
  if (rc != FBFFT_SUCCESS) return rc;
  if (!okArray(output, 4) || !sameShape(input, output)) return FBFFT_UNSUPPORTED_DIMENSION;
  if ((mean && !okStatistics(mean, input, groups)) || (rstd && !okStatistics(rstd, input, groups))) return FBFFT_UNSUPPORTED_DIMENSION;
  if (!(eps >= 0.f) || std::isinf(eps)) return FBFFT_UNSUPPORTED_SIZE;
  const long long pixels = input->size[2] * input->size[3];
  if (input->size[0] * input->size[1] * pixels == 0) return FBFFT_SUCCESS;
  if (!okWorkspace(workspace, workspaceBytes, fbfft_group_norm_workspace(0, input->size[0], input->size[1], pixels, groups)))
    return FBFFT_UNSUPPORTED_DIMENSION;
  NormProblem p = normOf(input, weight, bias, mean, rstd, groups, activation, workspace);
  p.y = imageOf(output);
  p.eps = eps;
  return launchNormForward(p, stream);
}

extern "C" int fbfft_group_norm_bprop(const fbfft_array* input, const fbfft_array* weight, const fbfft_array* bias,
                                      const fbfft_array* mean, const fbfft_array* rstd, const fbfft_array* gradOutput,
                                      const fbfft_array* gradInput, const fbfft_array* gradWeight,
                                      const fbfft_array* gradBias, long long groups, int activation, void* workspace,
                                      size_t workspaceBytes, fbfft_stream_t stream) {
  const int rc = checkNorm(input, weight, bias, groups, activation);
  if (rc != FBFFT_SUCCESS) return rc;
  const long long C = input->size[1];
  if (!okArray(gradOutput, 4) || !sameShape(input, gradOutput)) return FBFFT_UNSUPPORTED_DIMENSION;
  if (gradInput && (!okArray(gradInput, 4) || !sameShape(input, gradInput))) return FBFFT_UNSUPPORTED_DIMENSION;
  if (!okLine(gradWeight, C) || !okLine(gradBias, C)) return FBFFT_UNSUPPORTED_DIMENSION;
  if (!okStatistics(mean, input, groups) || !okStatistics(rstd, input, groups)) return FBFFT_UNSUPPORTED_DIMENSION;
  const long long pixels = input->size[2] * input->size[3];
  if (C == 0 || (!gradInput && !gradWeight && !gradBias)) return FBFFT_SUCCESS;
  if (!okWorkspace(workspace, workspaceBytes, fbfft_group_norm_workspace(1, input->size[0], C, pixels, groups)))
    return FBFFT_UNSUPPORTED_DIMENSION;
  NormProblem p = normOf(input, weight, bias, mean, rstd, groups, activation, workspace);
  p.g = imageOf(gradOutput), p.y = imageOf(gradInput);
  p.gradWeight = lineOf(gradWeight), p.gradBias = lineOf(gradBias);
  return launchNormBackward(p, stream);
}

extern "C" size_t fbfft_linear_workspace(int pass, long long M, long long K, long long N, int type) {
  if (pass < 0 || pass > 1 || M <= 0 || K < 0 || N <= 0 || type < FBFFT_FLOAT32 || type > FBFFT_BFLOAT16) return 0;
  if (M > kMost / N || (K > 0 && (M > kMost / K || N > kMost / K))) return 0;
  return linearWorkspaceBytes(pass, M, K, N, type);
}

namespace {
// (rows and columns by their number; what a launch can hold of their product is checked with the launch)
bool okLinearSize(long long n) { return n < 1ll << 23; }
}  // namespace

extern "C" int fbfft_linear_fprop(const fbfft_array* input, const fbfft_array* weight, const fbfft_array* bias,
                                  const fbfft_array* residual, const fbfft_array* output, const fbfft_array* preactivation,
                                  int activation, void* workspace, size_t workspaceBytes, fbfft_stream_t stream) {
  if (!okArray(input, 2) || !okArray(weight, 2) || !okActivation(activation)) return FBFFT_UNSUPPORTED_DIMENSION;
  const long long M = input->size[0], K = input->size[1], N = weight->size[0];
  const int type = input->type;
  if (!okMatrix(weight, N, K, type) || !okMatrix(output, M, N, type) || !okLine(bias, N)) return FBFFT_UNSUPPORTED_DIMENSION;
  if ((residual && !okMatrix(residual, M, N, type)) || (preactivation && !okMatrix(preactivation, M, N, type)))
    return FBFFT_UNSUPPORTED_DIMENSION;
  if (!okLinearSize(M) || !okLinearSize(N)) return FBFFT_UNSUPPORTED_SIZE;
  if (M == 0 || N == 0) return FBFFT_SUCCESS;
  if (!okWorkspace(workspace, workspaceBytes, fbfft_linear_workspace(0, M, K, N, type))) return FBFFT_UNSUPPORTED_DIMENSION;
  LinearProblem p{};
  p.x = matrixOf(input), p.w = matrixOf(weight), p.residual = matrixOf(residual), p.y = matrixOf(output), p.z = matrixOf(preactivation);
  p.bias = lineOf(bias);
  p.M = M, p.K = K, p.N = N, p.type = type, p.activation = activation, p.workspace = workspace;
  return launchLinearForward(p, stream);
}

extern "C" int fbfft_linear_bprop(const fbfft_array* input, const fbfft_array* weight, const fbfft_array* gradOutput,
                                  const fbfft_array* preactivation, const fbfft_array* gradInput,
                                  const fbfft_array* gradWeight, const fbfft_array* gradBias, int activation, void* workspace,
                                  size_t workspaceBytes, fbfft_stream_t stream) {
  if (!okArray(gradOutput, 2) || !okActivation(activation)) return FBFFT_UNSUPPORTED_DIMENSION;
  const long long M = gradOutput->size[0], N = gradOutput->size[1];
  const int type = gradOutput->type;
  const fbfft_array* named = weight ? weight : input ? input : gradInput ? gradInput : gradWeight;
  if (named && named->dim != 2) return FBFFT_UNSUPPORTED_DIMENSION;
  const long long K = named ? named->size[1] : 0;
  if ((gradInput && !weight) || (gradWeight && !input)) return FBFFT_UNSUPPORTED_DIMENSION;
  if ((weight && !okMatrix(weight, N, K, type)) || (input && !okMatrix(input, M, K, type))) return FBFFT_UNSUPPORTED_DIMENSION;
  if ((gradInput && !okMatrix(gradInput, M, K, type)) || (gradWeight && !okMatrix(gradWeight, N, K, type)))
    return FBFFT_UNSUPPORTED_DIMENSION;
  if (activation != FBFFT_ACTIVATION_NONE ? !preactivation : false) return FBFFT_UNSUPPORTED_DIMENSION;
  if (preactivation && !okMatrix(preactivation, M, N, type)) return FBFFT_UNSUPPORTED_DIMENSION;
  if (!okLine(gradBias, N)) return FBFFT_UNSUPPORTED_DIMENSION;
  if (!okLinearSize(M) || !okLinearSize(N) || !okLinearSize(K)) return FBFFT_UNSUPPORTED_SIZE;
  // (an operand that is not given has not been checked, and no size of a workspace stands for such products: 0 is that of
  // calls that need none)
  if (M * K > kMost || N * K > kMost) return FBFFT_UNSUPPORTED_SIZE;
  if (!okWorkspace(workspace, workspaceBytes, fbfft_linear_workspace(1, M, K, N, type))) return FBFFT_UNSUPPORTED_DIMENSION;
  LinearProblem p{};
  p.x = matrixOf(input), p.w = matrixOf(weight), p.dy = matrixOf(gradOutput), p.z = matrixOf(preactivation);
  p.dx = matrixOf(gradInput), p.dw = matrixOf(gradWeight), p.gradBias = lineOf(gradBias);
  p.M = M, p.K = K, p.N = N, p.type = type, p.activation = activation, p.workspace = workspace;
  return launchLinearBackward(p, stream);
}

namespace {

int dropoutOf(const fbfft_array* input, const fbfft_array* residual, const fbfft_array* output, double p,
              unsigned long long seed, unsigned long long offset, const unsigned long long* step, fbfft_stream_t stream) {
  if (!input || input->dim < 1 || input->dim > FBFFT_MAX_DIM) return FBFFT_UNSUPPORTED_DIMENSION;
  const int dim = input->dim;
  if (!okArray(input, dim) || !okArray(output, dim) || !sameShape(input, output)) return FBFFT_UNSUPPORTED_DIMENSION;
  if (residual && (!okArray(residual, dim) || !sameShape(input, residual))) return FBFFT_UNSUPPORTED_DIMENSION;
  if (!aligned(step, 8)) return FBFFT_UNSUPPORTED_DIMENSION;
  if (!(p >= 0.0 && p <= 1.0)) return FBFFT_UNSUPPORTED_SIZE;
  DropoutProblem d{};
  d.x = input->data, d.residual = residual ? residual->data : nullptr, d.y = output->data;
  d.total = 1;
  for (int i = 0; i < FBFFT_MAX_DIM; ++i) d.size[i] = 1;
  for (int i = 0; i < dim; ++i) {
    const int at = FBFFT_MAX_DIM - dim + i;
    d.size[at] = input->size[i];
    d.xs[at] = input->stride[i], d.ys[at] = output->stride[i], d.rs[at] = residual ? residual->stride[i] : 0;
    d.total *= input->size[i];
  }
  if (d.total == 0) return FBFFT_SUCCESS;
  d.type = input->type;
  d.threshold = (unsigned)std::floor(p * 65536.0 + 0.5);
  d.seed = seed, d.offset = offset, d.step = step;
  return launchDropout(d, stream);
}

}  // namespace

extern "C" int fbfft_dropout_fprop(const fbfft_array* input, const fbfft_array* residual, const fbfft_array* output, double p,
                                   unsigned long long seed, unsigned long long offset, const unsigned long long* step,
                                   fbfft_stream_t stream) {
  return dropoutOf(input, residual, output, p, seed, offset, step, stream);
}

extern "C" int fbfft_dropout_bprop(const fbfft_array* gradOutput, const fbfft_array* gradInput, double p,
                                   unsigned long long seed, unsigned long long offset, const unsigned long long* step,
                                   fbfft_stream_t stream) {
  return dropoutOf(gradOutput, nullptr, gradInput, p, seed, offset, step, stream);
}

extern "C" size_t fbfft_layer_norm_workspace(int pass, long long rows, long long cols) {
  if (pass < 0 || pass > 1 || rows <= 0 || cols <= 0 || rows > 0x7fffffff || cols > 0x7fffffff || rows > kMost / cols) return 0;
  return layerNormWorkspaceBytes(pass, rows, cols);
}

namespace {

bool okRowStatistics(const fbfft_array* a, long long rows) {
  return okArray(a, 1) && a->type == FBFFT_FLOAT32 && a->size[0] == rows;
}

// What both passes of layer norm share; 0 or an error.
int checkLayerNorm(const fbfft_array* input, const fbfft_array* weight) {
  if (!okArray(input, 2) || !okLine(weight, input->size[1])) return FBFFT_UNSUPPORTED_DIMENSION;
  return input->size[0] > 0x7fffffff || input->size[1] > 0x7fffffff ? FBFFT_UNSUPPORTED_SIZE : FBFFT_SUCCESS;
}

LayerNormProblem layerNormOf(const fbfft_array* input, const fbfft_array* weight, const fbfft_array* mean,
                             const fbfft_array* rstd, void* workspace) {
  LayerNormProblem p{};
  p.x = matrixOf(input), p.weight = lineOf(weight);
  if (mean) p.mean = static_cast<float*>(mean->data), p.meanStride = mean->stride[0];
  if (rstd) p.rstd = static_cast<float*>(rstd->data), p.rstdStride = rstd->stride[0];
  p.M = input->size[0], p.N = input->size[1], p.type = input->type, p.workspace = workspace;
  return p;
}

}  // namespace

extern "C" int fbfft_layer_norm_fprop(const fbfft_array* input, const fbfft_array* weight, const fbfft_array* bias,
                                      const fbfft_array* output, const fbfft_array* mean, const fbfft_array* rstd, float eps,
                                      void* workspace, size_t workspaceBytes, fbfft_stream_t stream) {
  const int rc = checkLayerNorm(input, weight);
  if (rc != FBFFT_SUCCESS) return rc;
  const long long M = input->size[0], N = input->size[1];
  if (!okMatrix(output, M, N, input->type) || !okLine(bias, N)) return FBFFT_UNSUPPORTED_DIMENSION;
  if ((mean && !okRowStatistics(mean, M)) || (rstd && !okRowStatistics(rstd, M))) return FBFFT_UNSUPPORTED_DIMENSION;
  if (!(eps >= 0.f) || std::isinf(eps)) return FBFFT_UNSUPPORTED_SIZE;
  if (M * N == 0) return FBFFT_SUCCESS;
  if (!okWorkspace(workspace, workspaceBytes, fbfft_layer_norm_workspace(0, M, N))) return FBFFT_UNSUPPORTED_DIMENSION;
  LayerNormProblem p = layerNormOf(input, weight, mean, rstd, workspace);
  p.y = matrixOf(output), p.bias = lineOf(bias), p.eps = eps;
  return launchLayerNormForward(p, stream);
}

extern "C" int fbfft_layer_norm_bprop(const fbfft_array* input, const fbfft_array* weight, const fbfft_array* mean,
                                      const fbfft_array* rstd, const fbfft_array* gradOutput, const fbfft_array* gradInput,
                                      const fbfft_array* gradWeight, const fbfft_array* gradBias, void* workspace,
                                      size_t workspaceBytes, fbfft_stream_t stream) {
  const int rc = checkLayerNorm(input, weight);
  if (rc != FBFFT_SUCCESS) return rc;
  const long long M = input->size[0], N = input->size[1];
  if (!okMatrix(gradOutput, M, N, input->type) || (gradInput && !okMatrix(gradInput, M, N, input->type)))
    return FBFFT_UNSUPPORTED_DIMENSION;
  if (!okLine(gradWeight, N) || !okLine(gradBias, N)) return FBFFT_UNSUPPORTED_DIMENSION;
  if (!okRowStatistics(mean, M) || !okRowStatistics(rstd, M)) return FBFFT_UNSUPPORTED_DIMENSION;
  if (N == 0 || (!gradInput && !gradWeight && !gradBias)) return FBFFT_SUCCESS;
  if (!okWorkspace(workspace, workspaceBytes, fbfft_layer_norm_workspace(1, M, N))) return FBFFT_UNSUPPORTED_DIMENSION;
  LayerNormProblem p = layerNormOf(input, weight, mean, rstd, workspace);
  p.g = matrixOf(gradOutput), p.y = matrixOf(gradInput);
  p.gradWeight = lineOf(gradWeight), p.gradBias = lineOf(gradBias);
  return launchLayerNormBackward(p, stream);
}

namespace {

constexpr long long kMostSide = 65536;  // of a matrix that is orthogonalised
constexpr double kMostSingular = 32;    // of what its products meet: pieces hold numbers below 64

// Whether singular values that start in [0, 1] and what the products make of them stay within kMostSingular under these
// polynomials: the greatest magnitude of each over the interval so far, at its ends and where its derivative is 0.
bool staysInside(const float* coefficients, int steps) {
  double most = 1;
  for (int i = 0; i < steps; ++i) {
    const double a = coefficients[3 * i], b = coefficients[3 * i + 1], c = coefficients[3 * i + 2];
    if (!std::isfinite(a) || !std::isfinite(b) || !std::isfinite(c)) return false;
    double next = 0, inner = 0;
    auto at = [&](double u) {  // u: the singular value's square
      if (!(u >= 0 && u <= most * most)) return;
      next = std::fmax(next, std::fabs(std::sqrt(u) * (a + u * (b + u * c))));
      inner = std::fmax(inner, std::fabs(u * (b + u * c)));
    };
    at(most * most);
    if (c != 0) at(-b / (2 * c));
    // a + 3 b u + 5 c u^2 = 0
    const double d = 9 * b * b - 20 * a * c;
    if (c == 0) {
      if (b != 0) at(-a / (3 * b));
    } else if (d >= 0) {
      at((-3 * b + std::sqrt(d)) / (10 * c));
      at((-3 * b - std::sqrt(d)) / (10 * c));
    }
    if (!(next <= kMostSingular && inner <= kMostSingular && most * most <= kMostSingular)) return false;
    most = next;
  }
  return true;
}

}  // namespace

extern "C" size_t fbfft_orthogonalize_workspace(long long batch, long long rows, long long cols) {
  if (batch <= 0 || rows <= 0 || cols <= 0 || rows > kMostSide || cols > kMostSide || batch > kMost / (rows * cols)) return 0;
  return orthogonalWorkspaceBytes(batch, rows, cols);
}

extern "C" int fbfft_orthogonalize(const fbfft_array* input, const fbfft_array* output, const float* coefficients, int steps,
                                   float eps, float scale, void* workspace, size_t workspaceBytes, fbfft_stream_t stream) {
  const int dim = input ? input->dim : 0;
  if ((dim != 2 && dim != 3) || !okArray(input, dim) || !okArray(output, dim) || !sameShape(input, output) || !coefficients)
    return FBFFT_UNSUPPORTED_DIMENSION;
  const long long batch = dim == 3 ? input->size[0] : 1, rows = input->size[dim - 2], cols = input->size[dim - 1];
  if (steps < 1 || steps > 32 || !(eps >= 0.f) || std::isinf(eps) || !std::isfinite(scale)) return FBFFT_UNSUPPORTED_SIZE;
  if (!staysInside(coefficients, steps)) return FBFFT_UNSUPPORTED_SIZE;
  if (batch * rows * cols == 0) return FBFFT_SUCCESS;
  if (rows > kMostSide || cols > kMostSide) return FBFFT_UNSUPPORTED_SIZE;
  if (!okWorkspace(workspace, workspaceBytes, fbfft_orthogonalize_workspace(batch, rows, cols))) return FBFFT_UNSUPPORTED_DIMENSION;
  OrthogonalProblem p{};
  p.x = Matrix{input->data, (long)input->stride[dim - 2], (long)input->stride[dim - 1]};
  p.y = Matrix{output->data, (long)output->stride[dim - 2], (long)output->stride[dim - 1]};
  if (dim == 3) p.xBatch = input->stride[0], p.yBatch = output->stride[0];
  p.batch = batch, p.rows = rows, p.cols = cols, p.type = input->type;
  p.coefficients = coefficients, p.steps = steps, p.eps = eps, p.scale = scale, p.workspace = workspace;
  return launchOrthogonalize(p, stream);
}

namespace {

constexpr long long kMostBlocks = 1 << 17;      // of a row in the 4-bit format
constexpr long long kMostCodeStride = 1 << 22;  // 256 of them are far inside 31 bits

bool okMx4(const fbfft_mx4* a) {
  if (!a || a->rows < 0 || a->blocks < 0 || a->rows > kMost || a->blocks > kMost) return false;
  if (a->rows == 0 || a->blocks == 0) return true;
  if (!a->codes || !a->scales || !aligned(a->codes, 16)) return false;
  return a->rows == 1 || (a->codeStride % 16 == 0 && a->codeStride >= 16 * a->blocks && a->scaleStride >= a->blocks);
}
bool okMx4Size(const fbfft_mx4* a) {
  return a->blocks <= kMostBlocks && (a->rows <= 1 || (a->codeStride <= kMostCodeStride && a->scaleStride <= kMostCodeStride));
}
Mx4 mx4Of(const fbfft_mx4* a) {
  if (!a) return Mx4{};
  const bool one = a->rows <= 1;  // (whose strides say nothing)
  return Mx4{static_cast<unsigned char*>(a->codes), static_cast<unsigned char*>(a->scales), (long)(one ? 16 * a->blocks : a->codeStride),
             (long)(one ? a->blocks : a->scaleStride)};
}

// whether `array` is rows that `packed` holds or is to hold
bool okPacked(const fbfft_array* array, const fbfft_mx4* packed) {
  return okArray(array, 2) && okMx4(packed) && packed->rows == array->size[0] && packed->blocks == (array->size[1] + 31) / 32;
}

}  // namespace

extern "C" int fbfft_mx4_quantize(const fbfft_array* input, const fbfft_mx4* output, fbfft_stream_t stream) {
  if (!okPacked(input, output)) return FBFFT_UNSUPPORTED_DIMENSION;
  const long long M = input->size[0], K = input->size[1];
  if (M > 0x7fffffff || !okMx4Size(output)) return FBFFT_UNSUPPORTED_SIZE;
  if (M * K == 0) return FBFFT_SUCCESS;
  return launchMx4Quantize(matrixOf(input), input->type, M, K, mx4Of(output), stream);
}

extern "C" int fbfft_mx4_dequantize(const fbfft_mx4* input, const fbfft_array* output, fbfft_stream_t stream) {
  if (!okPacked(output, input)) return FBFFT_UNSUPPORTED_DIMENSION;
  const long long M = output->size[0], K = output->size[1];
  if (M > 0x7fffffff || !okMx4Size(input)) return FBFFT_UNSUPPORTED_SIZE;
  if (M * K == 0) return FBFFT_SUCCESS;
  return launchMx4Dequantize(mx4Of(input), matrixOf(output), output->type, M, K, stream);
}

extern "C" size_t fbfft_linear_mx4_workspace(long long M, long long K, long long N) {
  if (M <= 0 || K < 0 || N <= 0 || !okLinearSize(M) || !okLinearSize(N) || K > kMostBlocks * 32) return 0;
  return linearMx4WorkspaceBytes(M, (K + 31) / 32, N);
}

extern "C" int fbfft_linear_mx4_fprop(const fbfft_array* input, const fbfft_mx4* quantized, const fbfft_mx4* weight,
                                      const fbfft_array* bias, const fbfft_array* residual, const fbfft_array* output,
                                      int activation, void* workspace, size_t workspaceBytes, fbfft_stream_t stream) {
  if (!okArray(output, 2) || !okMx4(weight) || !okActivation(activation) || !input == !quantized) return FBFFT_UNSUPPORTED_DIMENSION;
  const long long M = output->size[0], N = output->size[1], blocks = weight->blocks;
  const int type = output->type;
  if (weight->rows != N || !okLine(bias, N) || (residual && !okMatrix(residual, M, N, type))) return FBFFT_UNSUPPORTED_DIMENSION;
  if (input ? !okArray(input, 2) || input->type != type || input->size[0] != M || (input->size[1] + 31) / 32 != blocks
            : !okMx4(quantized) || quantized->rows != M || quantized->blocks != blocks)
    return FBFFT_UNSUPPORTED_DIMENSION;
  if (!okLinearSize(M) || !okLinearSize(N) || !okMx4Size(weight) || (quantized && !okMx4Size(quantized)))
    return FBFFT_UNSUPPORTED_SIZE;
  if (M == 0 || N == 0) return FBFFT_SUCCESS;
  if (!okWorkspace(workspace, workspaceBytes, fbfft_linear_mx4_workspace(M, 32 * blocks, N))) return FBFFT_UNSUPPORTED_DIMENSION;
  LinearMx4Problem p{};
  p.x = matrixOf(input), p.xq = mx4Of(quantized), p.w = mx4Of(weight);
  p.residual = matrixOf(residual), p.y = matrixOf(output), p.bias = lineOf(bias);
  p.M = M, p.K = input ? input->size[1] : 32 * blocks, p.blocks = blocks, p.N = N;
  p.type = type, p.activation = activation, p.workspace = workspace;
  return launchLinearMx4(p, stream);
}
