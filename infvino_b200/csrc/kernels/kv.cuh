// Host-visible declarations of the language-model kernels: rotary positions,
// the paged 8-bit key/value cache, and the attention over it.
#pragma once

#include <cstdint>
#include <cuda_runtime.h>

#include "conv_tc.cuh"  // FastDiv

namespace ivb {

constexpr int kKvBlock = 16;       // tokens that share a scale
constexpr int kKvMaxPairs = 128;   // rotated pairs of a head
constexpr int kKvMaxAxes = 4;
constexpr int kKvMinExp = -120, kKvMaxExp = 121;  // exponents of a scale: 2^e and 2^-e are normal floats

struct KvRows {       // 16-bit rows: element (token, head, d) at p[token * ts + head * hs + d]
  void *p;
  long long ts, hs;
  int vec;            // base and strides on 16 bytes
};

struct KvCache {
  int8_t *k, *v;      // [pages][heads][page][dim]
  float *ks, *vs;     // [pages][heads][page / kKvBlock]
  long long pages;
  int page, heads, dim;
};

struct KvSeqs {
  int batch;
  long long tokens;
  const int32_t *offsets, *at, *pages;
  int pps;            // pages per sequence (row length of `pages`)
};

struct KvRotary {
  const float2 *table;  // [positions][pairs] cos, sin; null: no rotation
  long long positions;
  int pairs, interleaved;
  const int32_t *pos[kKvMaxAxes];  // a token's positions on each axis (one that no pair turns by: another's again)
  uint32_t one_axis;    // bit g: the eight pairs 8g.. share an axis
  uint8_t axis[kKvMaxPairs];
};

struct KvAttend {
  KvCache cache;
  KvSeqs seqs;
  int q_heads, group, max_new;
  KvRows q, out;
  float scale;
  int window, sinks;
  int *status;
  FastDiv by_group, by_page;
  long long probe;  // above 0: every other CTA of the prompt kernel first waits so many SM clocks for what never comes
};

struct KvRopeFreq {
  double inv[kKvMaxPairs];
};
cudaError_t launch_kv_rope_table(const KvRopeFreq &freq, int pairs, long long positions, float2 *table, cudaStream_t st);
cudaError_t launch_kv_rope(bool bf16, long long tokens, int heads, int dim, const KvRows &x, const KvRows &out,
                           const KvRotary &rot, int *status, cudaStream_t st);
cudaError_t launch_kv_append(bool bf16, const KvCache &c, const KvSeqs &s, const KvRows &k, const KvRows &v,
                             const KvRotary &rot, int q_heads, const KvRows &q, const KvRows &q_out, int *status,
                             cudaStream_t st);
cudaError_t launch_kv_read(bool bf16, const KvCache &c, const KvSeqs &s, const KvRows &k, const KvRows &v, int *status,
                           cudaStream_t st);
// The workspace of a stream's attention calls: counters (zeroed once, they
// return to zero by themselves), then partial results.
constexpr size_t kKvCounterBytes = 1 << 14;
size_t kv_workspace_bytes(int sms);
size_t kv_prompt_workspace_bytes(int sms);  // the part that kv_prompt.cu needs
bool kv_prompt_takes(const KvAttend &a);
cudaError_t launch_kv_prompt(bool bf16, const KvAttend &a, void *workspace, int sms, cudaStream_t st);
cudaError_t launch_kv_attend(bool bf16, const KvAttend &a, void *workspace, int sms, cudaStream_t st);

}  // namespace ivb
