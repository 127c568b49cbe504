// spb_logprob_plan.h -- how a call of k_logprobs is cut: a row's parts, the CTAs that share them and the
// shared memory that keeps CTAs apart. Plain C++: the rule is checked without a GPU.
#pragma once

namespace spb {

constexpr int LPART = 16384;   // entries of a part, up to LPARTS parts
constexpr int LPARTS = 16;
constexpr int LPADS[3] = {0, 52 * 1024, 92 * 1024};   // unused shared memory: three, two, one CTA per SM

struct LogprobPlan {
  int parts, per;   // of a row, entries of a part: these follow from the vocabulary alone, and with them the bytes
  int ctas;         // of a row: a cluster
  int pad;          // unused dynamic shared memory of a CTA
};

// fits(ctas, pad): a cluster of that many CTAs with that much unused memory can run on the device. Where the
// wanted one cannot, it goes without the memory, then smaller: the results are the same.
template <typename Fits>
LogprobPlan plan_logprobs(int rows, int vocab, Fits &&fits) {
  int P = (vocab + LPART - 1) / LPART;
  if (P > LPARTS) P = LPARTS;
  const int per = ((vocab + P - 1) / P + 3) & ~3;
  P = (vocab + per - 1) / per;
  // few rows: a row over as many CTAs as it has parts; more: over fewer, so that the call is one wave of two
  // CTAs per SM (64 rows x 262144, 20 alternatives, at that step: 45 us with at most one per SM, 29 with two,
  // 43 and 61 with two and four waves); many rows: a CTA each, three per SM
  int C = P;
  if ((long long)rows * C > 2 * 148) C = rows < 2 * 148 ? 2 * 148 / rows : 1;
  for (;; C--) {
    const int each = (P + C - 1) / C;   // parts of a CTA, spread evenly
    C = (P + each - 1) / each;
    // calls of one wave spread over all SMs: unused shared memory keeps a second (third) CTA off an SM, where
    // the scheduler would fill it first (64 rows: 30 -> 26 us)
    const long long ctas = (long long)rows * C;
    const int pad = LPADS[ctas <= 148 ? 2 : ctas <= 2 * 148 ? 1 : 0];
    if (C == 1 || fits(C, pad)) return {P, per, C, pad};
    if (pad && fits(C, 0)) return {P, per, C, 0};
  }
}

}  // namespace spb
