// C ABI of the operators around a convolution layer: argument validation and dispatch.
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
