// logprobs.hip - log probabilities of given tokens, entropies and the top
// alternatives of rows of logits.
#include "common.h"

using namespace ihip;

struct LogprobArgs {
  const float* x;
  int64_t stride;
  const int* ids;
  float *logprobs, *entropy;
  int* top_ids;
  float* top_logprobs;
  int32_t rows, vocab, k, pad;
};

// a logit's place in the order of the alternatives: larger values first (both
// zeros the same), NaN behind -infinity; then the lower id
__device__ __forceinline__ uint32_t order_of(float v)
{
  if (v != v) return 0u;
  const uint32_t b = float_bits(v + 0.0f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

extern "C" __global__ __launch_bounds__(256) void logprobs(LogprobArgs a)
{
  const int r = blockIdx.x, t = threadIdx.x;
  const float* x = a.x + (int64_t)r * a.stride;
  __shared__ double red[8];
  __shared__ uint64_t best[4];
  float m = -__builtin_inff();
  bool nan = false;
  for (int i = t; i < a.vocab; i += 256) {
    m = fmaxf(m, x[i]);
    nan |= x[i] != x[i];
  }
  m = wave_max(m);
  if ((t & 63) == 0) red[t >> 6] = m;
  nan = __syncthreads_or(nan);
  m = fmaxf(fmaxf((float)red[0], (float)red[1]), fmaxf((float)red[2], (float)red[3]));
  __syncthreads();
  double s = 0, w = 0;
  for (int i = t; i < a.vocab; i += 256) {
    const float d = x[i] - m;
    const float e = expf(d);
    s += e;
    if (e > 0) w += (double)d * e;
  }
  s = wave_sum(s, 64);
  w = wave_sum(w, 64);
  if ((t & 63) == 0) {
    red[t >> 6] = s;
    red[4 + (t >> 6)] = w;
  }
  __syncthreads();
  s = red[0] + red[1] + red[2] + red[3];
  w = red[4] + red[5] + red[6] + red[7];
  const bool none = m == -__builtin_inff() && !nan;
  double ls = log(s);
  if (nan || m == __builtin_inff()) ls = __builtin_nan("");
  auto lp = [&](float v) { return none ? -__builtin_inff() : (float)((double)(v - m) - ls); };
  if (t == 0) {
    if (a.logprobs) {
      const int id = a.ids[r];
      a.logprobs[r] = id >= 0 && id < a.vocab ? lp(x[id]) : __builtin_nanf("");
    }
    if (a.entropy) a.entropy[r] = none ? 0.f : (float)(ls - w / s);
  }
  uint64_t last = ~0ull;
  for (int j = 0; j < a.k; j++) {
    uint64_t b = 0;
    for (int i = t; i < a.vocab; i += 256) {
      const uint64_t c = (uint64_t)order_of(x[i]) << 32 | (uint32_t)~i;
      if (c < last && c > b) b = c;
    }
    b = wave_max(b);
    __syncthreads();
    if ((t & 63) == 0) best[t >> 6] = b;
    __syncthreads();
    for (int i = 0; i < 4; i++) b = best[i] > b ? best[i] : b;
    last = b;
    if (t == 0) {
      const int id = j < a.vocab ? (int)~(uint32_t)b : -1;
      a.top_ids[(int64_t)r * a.k + j] = id;
      a.top_logprobs[(int64_t)r * a.k + j] = id >= 0 ? lp(x[id]) : -__builtin_inff();
    }
  }
}
