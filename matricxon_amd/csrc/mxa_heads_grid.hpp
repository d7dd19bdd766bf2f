// How heads_kernel's work is laid out over workgroups, in plain C++.
#pragma once

#include <algorithm>

#include "mxa_kv4_shape.hpp"

namespace mxa {

constexpr int kHeadThreads = 256;

struct HeadGrid {
  bool fast;  // whole vectors of 16 bytes
  int L;      // lanes of a head
  int TP;     // tokens of a workgroup
  int HQ, HK; // heads of q and of k of a workgroup: y has q's from y * HQ on, k's from y * HK on
  int split;  // grid.y; the last y has a head of q or of k, and so does every other
};

// qh heads of q and kh of k (cache: at least one, which divides qh), values of `size` bytes.
inline HeadGrid heads_grid(bool cache, int size, bool interleaved, int qh, int kh, int n_tokens, int dim, int rot) {
  HeadGrid g{};
  const int V = 16 / size, half = rot / 2;
  const int CR = interleaved ? rot / V : half / V, C = CR + (dim - rot) / V;
  g.fast = (interleaved ? rot : half) % V == 0 && (dim - rot) % V == 0 && C <= 64;
  g.L = 64;
  if (g.fast)
    for (g.L = 1; g.L < C;) g.L *= 2;
  const int per = kHeadThreads / g.L, W = kv_groups(dim), H = qh + kh;
  const auto shares = [](int n, int of) { return of > 0 ? (n + of - 1) / of : 0; };
  if (cache) {
    // One token a workgroup while that fills the CUs: 256 tokens 8.3 us (four: 9.7), 512 tokens 11.0 (10.3). Key heads then by
    // four (16 tokens, 32 + 8 heads: 6.6 us; eight 8.7, one 6.7 but 29 for 512 tokens); with four tokens sixteen groups, or
    // thirty-two where the call has 80000 groups of keys and more (some five workgroups of sixteen a CU), when a workgroup's
    // start is shared by more. us of a captured call, sixteen and thirty-two: 32 + 8 heads of 128, 2048 tokens 17.3 and 18.4,
    // 2500 21.7 and 21.5, 3500 27.5 and 25.1, 8192 49 and 43; 64 + 16 of 64 the same; 16 + 8 of 256, 1024 tokens 14.8 and 15.4,
    // 1536 21.3 and 19.0, 4096 44.9 and 38.9.
    g.TP = n_tokens > 256 ? 4 : 1;
    const int room = std::max(1, 8192 / (g.TP * 32 * W));  // keys that 32 KB hold
    g.HK = std::min(std::min(kh, room), g.TP == 1 ? 4 : std::max(1, ((long long)n_tokens * kh * W >= 80000 ? 32 : 16) / W));
    g.HQ = g.HK * (qh / kh);
  } else {
    // tokens share what their sines cost; up to 512 the heads of one are spread over workgroups instead
    g.TP = n_tokens > 512 ? std::min(8, (n_tokens + 1023) / 1024) : 1;
    const int split = n_tokens > 512 ? 1 : std::min(4096, (H + per - 1) / per);
    g.HQ = shares(qh, split);
    g.HK = shares(kh, split);
  }
  // Both shares are rounded up, so that fewer workgroups than the shares were made for may have them all: 64 + 8 heads by nine
  // are 8 and 1 for each of eight, and a ninth would begin behind the last head.
  g.split = std::max(shares(qh, g.HQ), shares(kh, g.HK));
  return g;
}

}  // namespace mxa
