// Launchers of lm_loss.hip: losses and records over rows of vocabulary logits.
#pragma once

#include <hip/hip_runtime.h>
#include <cstdint>

enum LmType { LM_BF16 = 0, LM_FP16 = 1, LM_FP32 = 2 };

// R = B*T rows of V logits each; row r starts at x + (r/T)*sb + (r%T)*st
// elements, its logits lie side by side, at any alignment of one element.
struct LmRows {
  const void* x;
  long long sb, st;
  int T, R, V;
  int type;
  float c;           // log2(e) / temperature
  float c_hi, c_lo;  // the same in two parts, both positive
};

// What the backward pass keeps of a row: base gradient coef * w * 2^((x-mb)c),
// and at the places, coef * (mass_S * 2^((x-M)c) - p), where mass_S is the
// target's mass (1) over S.
struct LmStat {
  float mb, w, M, mass_S;
};

// The rows that count, and the places that get a gradient of their own.
struct LmPlaces {
  const void* idx;      // [R, K] int64 or int32
  const uint8_t* mask;  // [R] or null: 0 = the row is ignored
  long long ignore;     // K == 1: the row is ignored where idx == ignore
  int K, idx64, use_ignore;
};

// What the forward pass keeps for the backward one.
struct LmKeep {
  LmStat* stat;  // [R]
  float* coef;   // [R]; 0: the row has no gradient
  float* inv;    // 1 / rows that count, for a mean
  float* p;      // [R, K] a record's probabilities, or null: one place with 1
};

// Workspaces of one forward pass.
struct LmWork {
  int splits, group;        // blocks of a row, and lanes that join them
  float2 *part, *part_top;  // [R, splits]; part_top only where a record has a rest
  float* xt;                // [R], the logit of a loss's one place
  double4* rec;             // [R], distillation only
  double2* bpart;           // one per block of the finish kernel
  int* counter;
};

enum LmReduction { LM_MEAN = 0, LM_SUM = 1, LM_NONE = 2 };
struct LmOut {
  float* loss;  // [1], or one per row or pair
  float* inv;
  int reduction;
};

// The loss's upstream gradient: one, one per row, or one per pair of sequences.
enum LmUpPer { LM_UP_ALL = 0, LM_UP_ROW = 1, LM_UP_PAIR = 2 };
struct LmUp {
  const float* g;
  int per, pairs;
};

struct LmTeacher {
  const void* values;  // [R, K] of `type`
  const float* lse;    // [R], or null: the record is renormalised
  int type;
  double temperature;
};

struct LmPolicy {
  const float *old_lp, *adv, *ref_lp;  // [R]; ref_lp may be null
  double clip_low, clip_high, kl_coef;
};

struct LmPreference {
  const void* ref;  // [2 * pairs] float or double
  int ref64;
  double beta, smoothing;
};

constexpr int kLmMostK = 256;

int lm_stats_splits(const LmRows& in);
int lm_grad_splits(const LmRows& in);
int lm_group(int splits);
int lm_finish_blocks(int R, int group);

void lm_distill(const LmRows& in, const LmPlaces& pl, const LmTeacher& te,
                const LmWork& w, const LmKeep& kp, const LmOut& o,
                hipStream_t s);
void lm_policy(const LmRows& in, const LmPlaces& pl, const LmPolicy& po,
               const LmWork& w, const LmKeep& kp, float* logps, float* kl,
               const LmOut& o, hipStream_t s);
void lm_preference(const LmRows& in, const LmPlaces& pl, const LmPreference& pr,
                   const LmWork& w, const LmKeep& kp, float* chosen,
                   float* rejected, const LmOut& o, hipStream_t s);
// dx: [R, V], side by side
void lm_grad(const LmRows& in, const LmPlaces& pl, const LmKeep& kp,
             const LmUp& up, void* dx, hipStream_t s);
void lm_topk(const LmRows& in, double temperature, int k, void* values,
             long long* indices, float* lse, hipStream_t s);
