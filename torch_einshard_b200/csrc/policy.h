// Clipped policy loss with a KL term from logits (policy.cu).  dtype codes as in gemm.h.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace es {

enum PolicyReduction : int { kReduceMean = 0, kReduceSequence = 1, kReduceSum = 2 };

struct PolicyArgs {
  int dtype = 0;
  const void* logits = nullptr;  // [tokens, vocab], row pitch ld
  long long ld = 0, tokens = 0, vocab = 0;
  long long length = 1;            // tokens of a sequence (tokens = sequences * length)
  const int64_t* ids = nullptr;    // [tokens]
  const bool* mask = nullptr;      // [tokens]; null: every token counts
  const float* old = nullptr;      // [tokens]; null: the log-probabilities themselves
  const float* ref = nullptr;      // [tokens]; null: no KL term
  const float* adv = nullptr;      // [tokens], or one a sequence
  int adv_per_sequence = 0;
  double least = 0.8, most = 1.2;  // the clip range
  double kl = 0.0, inv_temp = 1.0;
  float weight = 1.0f;             // factor of the loss
  int reduction = kReduceMean;
  int sms = 148;
};

struct PolicySums {
  double loss, kl, clipped;
};

struct PolicyState {
  float* logp = nullptr;    // [tokens] output: log-probability of the token, 0 where masked
  float4* terms = nullptr;  // [tokens] logit, largest logit, sum of powers, derivative of the loss by logp (without weights)
  float* share = nullptr;   // [sequences] a token's share in the reduction, where the mask decides it
  PolicySums* sums = nullptr;  // [policy_sum_blocks] scratch
  unsigned* done = nullptr;    // scratch: blocks that are done
  float* loss = nullptr;    // scalars
  float* kl = nullptr;
  float* clipped = nullptr;
  // the gradient for an upstream gradient of `factors`: written by the forward pass (factors 1) where not null
  void* dlogits = nullptr;  // [tokens, vocab] contiguous
  float* factors = nullptr; // [tokens]
};

// Blocks that add the tokens' terms.
long long policy_sum_blocks(long long tokens);
int policy_forward(const PolicyArgs& a, const PolicyState& s, cudaStream_t stream, int* launches);
// s.dlogits for the gradient *grad of the loss.  With s.factors, rows that hold it already are left.
int policy_backward(const PolicyArgs& a, const PolicyState& s, const float* grad, cudaStream_t stream);

}  // namespace es
