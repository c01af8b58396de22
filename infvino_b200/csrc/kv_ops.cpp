// C ABI of the language-model operators (include/infvino_b200.h, ivc_kv_*):
// argument checks, the per-stream workspaces and the status word.  Exceptions
// never cross the boundary.
#include <algorithm>
#include <cstring>
#include <iterator>
#include <map>
#include <mutex>
#include <stdexcept>
#include <string>
#include <thread>
#include <utility>

#include "../../include/infvino_b200.h"
#include "kernels/common.cuh"
#include "kernels/kv.cuh"
#include "kernels/mx4.cuh"
#include "kernels/sample.cuh"

struct ivc_kv {
  int device = 0, sms = 0;
  mutable std::mutex mu;
  std::string err;                              // of the last failed call,
  std::map<std::thread::id, std::string> errs;  // and of each thread's
  int *status = nullptr;
  long long probe = 0;
  std::map<unsigned long long, void *> workspace;  // by the stream's id
  std::map<std::pair<cudaStream_t, std::thread::id>, unsigned long long> named;  // ids by handle value (and thread, for cudaStreamPerThread)
};

namespace {

thread_local std::string g_kv_create_err;
thread_local std::string g_kv_shown_err;  // what this thread's ivc_kv_last_error has returned: no other thread writes it

// The handle's device for the length of a call, and launches with programmatic
// dependent launch whatever an engine on this thread last chose.
class Scope {
 public:
  explicit Scope(int device) : pdl_(ivb::g_launch_pdl) {
    ivb::g_launch_pdl = true;
    if (cudaGetDevice(&before_) != cudaSuccess) before_ = device;
    if (before_ != device) changed_ = cudaSetDevice(device) == cudaSuccess;
  }
  ~Scope() {
    ivb::g_launch_pdl = pdl_;
    if (changed_) (void)cudaSetDevice(before_);
  }

 private:
  bool pdl_, changed_ = false;
  int before_ = 0;
};

struct Bad : std::runtime_error {
  using std::runtime_error::runtime_error;
};
struct CudaError : std::runtime_error {
  using std::runtime_error::runtime_error;
};
void need(bool ok, const char *what) {
  if (!ok) throw Bad(what);
}
void cuda(cudaError_t e, const char *what) {
  if (e == cudaSuccess) return;
  (void)cudaGetLastError();
  throw CudaError(std::string(what) + ": " + cudaGetErrorString(e));
}

// Runs f on the handle's device; what it throws becomes a status and a message.
template <class F>
int attempt(ivc_kv *h, std::string &why, F &&f) {
  int code = IVC_ERR_CUDA;
  try {
    Scope scope(h->device);
    f();
    return IVC_OK;
  } catch (const Bad &e) {
    code = IVC_ERR_ARGUMENT;
    why = e.what();
  } catch (const std::exception &e) {
    why = e.what();
  } catch (...) {
    why = "unknown error";
  }
  return code;
}

// (under the handle's lock)
void note(ivc_kv *h, const char *call, const std::string &why) {
  try {
    h->err = std::string(call) + ": " + why;
    h->errs[std::this_thread::get_id()] = h->err;
  } catch (...) {
  }
}

template <class F>
int guarded(ivc_kv *h, const char *call, F &&f) {
  if (!h) return IVC_ERR_ARGUMENT;
  std::lock_guard<std::mutex> lk(h->mu);
  std::string why;
  const int code = attempt(h, why, f);
  if (code != IVC_OK) note(h, call, why);
  return code;
}

// A stream's id tells it apart from others that run at the same time.  The
// handle's value does not: cudaStreamPerThread is one value for a stream of every
// thread, and a destroyed stream's value may be given out again while its work is
// pending.  A stream that is being captured does not tell its id; it is the one
// that its name stood for at the last call outside a capture (~0: none yet).  The
// legacy stream is never captured, and while others are it cannot be asked.
struct StreamName {
  unsigned long long &id;
  bool captured;
};
StreamName stream_name(ivc_kv *h, cudaStream_t st) {
  constexpr unsigned long long kLegacy = ~1ull;
  if (st == cudaStreamLegacy) st = nullptr;
  const auto name = std::make_pair(st, st == cudaStreamPerThread ? std::this_thread::get_id() : std::thread::id());
  unsigned long long &id = h->named.emplace(name, st ? ~0ull : kLegacy).first->second;
  if (!st) return {id, false};
  cudaStreamCaptureStatus cap = cudaStreamCaptureStatusNone;
  cuda(cudaStreamIsCapturing(st, &cap), "stream");
  const bool captured = cap != cudaStreamCaptureStatusNone;
  if (!captured) cuda(cudaStreamGetId(st, &id), "stream");
  return {id, captured};
}

// The stream's attention workspace, allocated and zeroed (in the stream's order) at its first use.
void *workspace(ivc_kv *h, cudaStream_t st) {
  const StreamName name = stream_name(h, st);
  const auto it = h->workspace.find(name.id);
  if (it != h->workspace.end()) return it->second;
  need(!name.captured, "a stream's first call cannot be captured: call ivc_kv_reserve before");
  const size_t bytes = ivb::kv_workspace_bytes(h->sms);
  void *p = nullptr;
  cuda(cudaMalloc(&p, bytes), "workspace");
  try {
    cuda(cudaMemsetAsync(p, 0, ivb::kKvCounterBytes, st), "workspace");
    h->workspace[name.id] = p;
  } catch (...) {
    (void)cudaFree(p);
    throw;
  }
  return p;
}

bool aligned(const void *p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

// Launch grids count tokens in 32 bits, and a row index times 16 threads stays inside them too.
constexpr int64_t kMaxTokens = 1 << 26;

ivb::KvRows rows(const ivc_rows *r, const char *what, int64_t tokens, int heads) {
  need(r != nullptr && (r->data != nullptr || tokens == 0), what);
  need(aligned(r->data, 2), "rows are 2-byte aligned");
  ivb::KvRows k;
  k.p = r->data;
  // the stride of an axis with one entry is never used
  k.ts = tokens > 1 ? r->token_stride : 0;
  k.hs = heads > 1 ? r->head_stride : 0;
  k.vec = aligned(r->data, 16) && k.ts % 8 == 0 && k.hs % 8 == 0;
  return k;
}

// Rows that are written: no two may share elements.
ivb::KvRows out_rows(const ivc_rows *r, const char *what, int64_t tokens, int heads, int dim) {
  const ivb::KvRows k = rows(r, what, tokens, heads);
  need((tokens <= 1 || k.ts >= dim || k.ts <= -dim) && (heads <= 1 || k.hs >= dim || k.hs <= -dim),
       "rows that are written overlap");
  return k;
}

void check_dtype(int dtype) { need(dtype == IVC_F16 || dtype == IVC_BF16, "dtype is IVC_F16 or IVC_BF16"); }

ivb::KvRotary rotation(const ivc_rotary *r, int head_dim, int64_t tokens) {
  ivb::KvRotary k;
  std::memset(&k, 0, sizeof(k));
  if (!r) return k;
  need(r->table && aligned(r->table, 16), "the rotary table is 16-byte aligned device memory");
  need(r->positions > 0, "the rotary table has no positions");
  need(r->pairs > 0 && r->pairs % 8 == 0 && r->pairs <= IVC_KV_MAX_PAIRS && 2 * r->pairs <= head_dim,
       "rotary pairs: a multiple of 8, and 2 * pairs at most head_dim");
  need(r->axes >= 1 && r->axes <= ivb::kKvMaxAxes, "rotary axes: 1 to 4");
  need(r->pos || tokens == 0, "no rotary positions");
  need(aligned(r->pos, 4), "rotary positions are int32");
  k.table = reinterpret_cast<const float2 *>(r->table);
  k.positions = r->positions;
  k.pairs = r->pairs;
  k.interleaved = r->interleaved != 0;
  for (int i = 0; i < r->pairs; ++i) {
    const int a = r->axis_of ? r->axis_of[i] : 0;
    need(a < r->axes, "axis_of names an axis that the positions lack");
    k.axis[i] = (uint8_t)a;
  }
  for (int a = 0; a < ivb::kKvMaxAxes; ++a) {
    const bool used = std::find(k.axis, k.axis + r->pairs, a) != k.axis + r->pairs;
    k.pos[a] = r->pos + (used ? a : k.axis[0]) * (r->axes > 1 ? r->pos_stride : 0);
  }
  for (int g = 0; g < r->pairs / 8; ++g) {
    bool one = true;
    for (int i = 1; i < 8; ++i) one = one && k.axis[8 * g + i] == k.axis[8 * g];
    if (one) k.one_axis |= 1u << g;
  }
  return k;
}

ivb::KvCache check_cache(const ivc_kv_cache *c) {
  need(c != nullptr, "no cache");
  need(c->k && c->v && c->k_scale && c->v_scale, "the cache has a null pointer");
  need(aligned(c->k, 16) && aligned(c->v, 16), "cache codes are 16-byte aligned");
  need(aligned(c->k_scale, 4) && aligned(c->v_scale, 4), "cache scales are float");
  need(c->pages > 0 && c->pages <= 0x7fffffffLL, "cache pages: 1 to 2^31 - 1");
  need(c->page_size > 0 && c->page_size % IVC_KV_BLOCK == 0 && c->page_size <= (1 << 20),
       "page_size is a multiple of IVC_KV_BLOCK");
  need(c->kv_heads > 0 && c->kv_heads <= 256, "kv_heads: 1 to 256");
  need(c->head_dim == 64 || c->head_dim == 128, "the cache's head_dim is 64 or 128");
  return ivb::KvCache{c->k, c->v, c->k_scale, c->v_scale, c->pages, c->page_size, c->kv_heads, c->head_dim};
}

ivb::KvSeqs check_seqs(const ivc_kv_seqs *s) {
  need(s != nullptr, "no sequences");
  need(s->batch >= 0 && s->batch <= (1 << 20), "batch out of range");
  need(s->tokens >= 0 && s->tokens <= kMaxTokens, "tokens out of range");
  need(s->batch > 0 || s->tokens == 0, "tokens without a sequence");
  need(s->batch == 0 || (s->offsets && s->at && s->pages), "the sequences have a null pointer");
  need(aligned(s->offsets, 4) && aligned(s->at, 4) && aligned(s->pages, 4), "offsets, at and pages are int32");
  need(s->pages_per_seq >= 1 || s->batch == 0, "pages_per_seq is at least 1");
  return ivb::KvSeqs{s->batch, s->tokens, s->offsets, s->at, s->pages, s->pages_per_seq};
}

ivb::KvAttend attention(const ivc_kv *h, const ivc_kv_cache *cache, const ivc_kv_seqs *seqs, int q_heads, int max_new,
                        const ivc_rows *q, const ivc_rows *out, float scale, int window, int sinks) {
  ivb::KvAttend a{};
  a.cache = check_cache(cache);
  a.seqs = check_seqs(seqs);
  need(q_heads > 0 && q_heads <= 65536 && q_heads % a.cache.heads == 0, "q_heads is a multiple of kv_heads");
  need(max_new >= 0 && (max_new > 0 || a.seqs.tokens == 0), "max_new is at least 1");
  need(window >= 0 && sinks >= 0, "window and sinks are not negative");
  a.q = rows(q, "q is null", a.seqs.tokens, q_heads);
  a.out = out_rows(out, "out is null", a.seqs.tokens, q_heads, a.cache.dim);
  a.q_heads = q_heads;
  a.group = q_heads / a.cache.heads;
  a.max_new = max_new;
  a.scale = scale;
  a.window = window;
  a.sinks = sinks;
  a.status = h->status;
  a.probe = h->probe;
  need((int64_t)max_new * a.group < (1LL << 30), "max_new * q_heads / kv_heads out of range");
  a.by_group = ivb::make_fastdiv((uint32_t)a.group);
  a.by_page = ivb::make_fastdiv((uint32_t)a.cache.page);
  return a;
}

ivb::Mx4 check_mx4(const ivc_mx4 *m) {
  need(m != nullptr, "no 4-bit matrix");
  need(m->rows >= 0 && m->rows <= 0x7fffffffLL, "rows of a 4-bit matrix: at most 2^31 - 1");
  need(m->width > 0 && m->width % IVC_MX4_BLOCK == 0 && m->width <= (1 << 24), "width of a 4-bit matrix: a multiple of IVC_MX4_BLOCK");
  need(m->rows == 0 || (m->codes && m->scales), "a 4-bit matrix has a null pointer");
  need(aligned(m->codes, 16) && aligned(m->scales, 16), "codes and scales are 16-byte aligned");
  return ivb::Mx4{m->codes, m->scales, m->rows, m->width};
}

// Memory that a call reads or writes: n pieces of `bytes` each, `stride` bytes apart.
struct Memory {
  int64_t at, n, stride, bytes;
  Memory(const void *p, int64_t count, int64_t apart, int64_t each)
      : at((int64_t)reinterpret_cast<uintptr_t>(p)), n(each > 0 ? count : 0), stride(count > 1 ? apart : 0), bytes(each) {
    if (stride < 0) at += stride * (n - 1), stride = -stride;
  }
  Memory(const void *p, int64_t all) : Memory(p, 1, 0, all) {}
  int64_t end() const { return at + stride * (n - 1) + bytes; }
};
// Whether one of m's pieces has a byte of lo .. hi - 1.
bool meets(const Memory &m, int64_t lo, int64_t hi) {
  // the first piece that ends behind lo
  const int64_t i = m.at + m.bytes > lo || m.stride == 0 ? 0 : (lo - m.bytes - m.at) / m.stride + 1;
  return i < m.n && m.at + i * m.stride + m.bytes > lo && m.at + i * m.stride < hi;
}
// Rows that lie between one another (columns of one buffer) do not meet.
bool meet(const Memory &a, const Memory &b) {
  if (a.n == 0 || b.n == 0 || a.end() <= b.at || b.end() <= a.at) return false;
  const Memory &few = a.n < b.n ? a : b, &many = a.n < b.n ? b : a;
  if (few.stride == many.stride) {  // (as the rows of the one, seen from every row of the other)
    Memory all = many;
    all.at -= few.stride * (few.n - 1);
    all.n += few.n - 1;
    return meets(all, few.at, few.at + few.bytes);
  }
  for (int64_t i = 0; i < few.n; ++i)
    if (meets(many, few.at + i * few.stride, few.at + i * few.stride + few.bytes)) return true;
  return false;
}

Memory codes_of(const ivb::Mx4 &m) { return Memory(m.codes, m.rows * (m.width / 2)); }
Memory scales_of(const ivb::Mx4 &m) { return Memory(m.scales, (m.rows + 127) / 128 * ((m.width + 127) / 128) * 512); }
Memory matrix(const void *p, int64_t rows, int64_t width, int64_t stride) { return Memory(p, rows, 2 * stride, 2 * width); }
ivb::Mx4 first_rows(ivb::Mx4 m, int64_t rows) { return m.rows = rows, m; }
bool apart(const Memory &a, const ivb::Mx4 &m) { return !meet(a, codes_of(m)) && !meet(a, scales_of(m)); }
bool apart(const ivb::Mx4 &a, const ivb::Mx4 &b) { return apart(codes_of(a), b) && apart(scales_of(a), b); }

// Whether rows of [tokens][heads][dim] meet m.
bool meet(const ivb::KvRows &r, int64_t tokens, int heads, int dim, const Memory &m) {
  const Memory head(r.p, tokens, 2 * r.ts, 2 * dim);
  const int64_t span = 2 * r.hs * (heads - 1);
  if (head.end() + std::max<int64_t>(span, 0) <= m.at || m.end() <= head.at + std::min<int64_t>(span, 0)) return false;
  for (int h = 0; h < heads; ++h) {
    Memory one = head;
    one.at += 2 * r.hs * h;
    if (meet(one, m)) return true;
  }
  return false;
}

void check_matrix(int dtype, const void *p, int64_t rows, int64_t width, int64_t stride, bool written) {
  check_dtype(dtype);
  need(rows >= 0 && rows <= kMaxTokens, "rows out of range");
  need(p != nullptr || rows == 0, "a matrix is null");
  need(aligned(p, 2), "rows are 2-byte aligned");
  need(!written || rows <= 1 || stride >= width || stride <= -width, "rows that are written overlap");
}

}  // namespace

extern "C" {

int ivc_kv_create(int device_ordinal, ivc_kv **out) {
  if (!out) return IVC_ERR_ARGUMENT;
  *out = nullptr;
  ivc_kv *h = nullptr;
  int code = IVC_ERR_CUDA;
  std::string why;
  try {
    int n = 0, major = 0;
    cuda(cudaGetDeviceCount(&n), "device count");
    need(device_ordinal >= 0 && device_ordinal < n, "no such device");
    cuda(cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, device_ordinal), "device attribute");
    need(major == 10, "the kernels are built for sm_100a");
    h = new ivc_kv;
    h->device = device_ordinal;
    cuda(cudaDeviceGetAttribute(&h->sms, cudaDevAttrMultiProcessorCount, device_ordinal), "device attribute");
    Scope scope(device_ordinal);
    cuda(cudaMalloc(&h->status, sizeof(int)), "status word");
    // Zero before any stream's kernel can set it: in a stream of its own, for the
    // legacy stream's order means nothing to streams that do not block.
    cudaStream_t st = nullptr;
    cuda(cudaStreamCreateWithFlags(&st, cudaStreamNonBlocking), "status word");
    cudaError_t e = cudaMemsetAsync(h->status, 0, sizeof(int), st);
    if (e == cudaSuccess) e = cudaStreamSynchronize(st);
    (void)cudaStreamDestroy(st);
    cuda(e, "status word");
    *out = h;
    return IVC_OK;
  } catch (const Bad &e) {
    code = IVC_ERR_ARGUMENT;
    why = e.what();
  } catch (const std::exception &e) {
    why = e.what();
  }
  ivc_kv_destroy(h);
  try {
    g_kv_create_err = "ivc_kv_create: " + why;
  } catch (...) {
  }
  return code;
}

void ivc_kv_destroy(ivc_kv *h) {
  if (!h) return;
  {
    Scope scope(h->device);
    for (auto &w : h->workspace) (void)cudaFree(w.second);  // (waits for the device)
    if (h->status) (void)cudaFree(h->status);
    (void)cudaGetLastError();
  }
  delete h;
}

const char *ivc_kv_last_error(const ivc_kv *h) {
  if (!h) return g_kv_create_err.c_str();
  std::lock_guard<std::mutex> lk(h->mu);
  try {
    const auto it = h->errs.find(std::this_thread::get_id());
    g_kv_shown_err = it != h->errs.end() ? it->second : h->err;
  } catch (...) {
    return "";
  }
  return g_kv_shown_err.c_str();
}

int ivc_kv_synchronize(ivc_kv *h, void *stream) {
  if (!h) return IVC_ERR_ARGUMENT;
  int word = 0;
  std::string why;
  // (not under the handle's lock: other threads' calls need not wait for this stream)
  int r = attempt(h, why, [&] {
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    cuda(cudaMemcpyAsync(&word, h->status, sizeof(int), cudaMemcpyDeviceToHost, st), "status word");
    cuda(cudaStreamSynchronize(st), "synchronize");
    if (word) {
      cuda(cudaMemsetAsync(h->status, 0, sizeof(int), st), "status word");
      cuda(cudaStreamSynchronize(st), "synchronize");
    }
  });
  if (r == IVC_OK && word != 0) {
    r = IVC_ERR_KERNEL;
    why = std::string(word == 16   ? "a page number outside the cache"
                      : word == 17 ? "offsets, positions or lengths that do not fit the call"
                      : word == 18 ? "a position outside the rotary table"
                                   : "a kernel's bounded wait timed out") +
          " (status " + std::to_string(word) + ")";
  }
  if (r != IVC_OK) {
    std::lock_guard<std::mutex> lk(h->mu);
    note(h, "ivc_kv_synchronize", why);
  }
  return r;
}

int ivc_kv_reserve(ivc_kv *h, void *stream) {
  return guarded(h, "ivc_kv_reserve", [&] { workspace(h, static_cast<cudaStream_t>(stream)); });
}

int ivc_kv_release(ivc_kv *h, void *stream) {
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  void *p = nullptr;
  const int r = guarded(h, "ivc_kv_release", [&] {
    const StreamName name = stream_name(h, st);
    need(!name.captured, "a stream that is being captured keeps its workspace");
    const unsigned long long id = name.id;
    const auto it = h->workspace.find(id);
    if (it == h->workspace.end()) return;
    p = it->second;
    h->workspace.erase(it);
    for (auto n = h->named.begin(); n != h->named.end();) n = n->second == id ? h->named.erase(n) : std::next(n);
  });
  if (!p) return r;
  // (not under the handle's lock: other threads' calls need not wait for this stream)
  Scope scope(h->device);
  (void)cudaStreamSynchronize(st);
  (void)cudaFree(p);
  (void)cudaGetLastError();
  return r;
}

int ivc_debug_kv_probe(ivc_kv *h, long long limit_cycles) {
  return guarded(h, "ivc_debug_kv_probe", [&] {
    need(limit_cycles >= 0 && limit_cycles <= ivb::kConvWaitLimitDefault, "the limit is from 0 to that of the other waits");
    h->probe = limit_cycles;
  });
}

int ivc_kv_rope_table(ivc_kv *h, const double *inv_freq, int pairs, int64_t positions, float *table, void *stream) {
  return guarded(h, "ivc_kv_rope_table", [&] {
    need(inv_freq && table, "null pointer");
    need(aligned(table, 16), "the rotary table is 16-byte aligned device memory");
    need(pairs > 0 && pairs <= IVC_KV_MAX_PAIRS, "rotary pairs: 1 to 128");
    need(positions > 0 && positions <= (1LL << 40), "positions out of range");
    ivb::KvRopeFreq f{};
    for (int i = 0; i < pairs; ++i) f.inv[i] = inv_freq[i];
    cuda(ivb::launch_kv_rope_table(f, pairs, positions, reinterpret_cast<float2 *>(table),
                                   static_cast<cudaStream_t>(stream)),
         "launch");
  });
}

int ivc_kv_rope(ivc_kv *h, int dtype, int64_t tokens, int heads, int head_dim, const ivc_rows *x, const ivc_rows *out,
                const ivc_rotary *rotary, void *stream) {
  return guarded(h, "ivc_kv_rope", [&] {
    check_dtype(dtype);
    need(tokens >= 0 && tokens <= kMaxTokens, "tokens out of range");
    need(heads > 0 && heads <= 65536, "heads out of range");
    need(head_dim > 0 && head_dim % 16 == 0 && head_dim <= 256, "head_dim: a multiple of 16, at most 256");
    need(rotary != nullptr, "no rotary");
    const ivb::KvRotary rot = rotation(rotary, head_dim, tokens);
    const ivb::KvRows a = rows(x, "x is null", tokens, heads), b = out_rows(out, "out is null", tokens, heads, head_dim);
    if (tokens == 0) return;
    cuda(ivb::launch_kv_rope(dtype == IVC_BF16, tokens, heads, head_dim, a, b, rot, h->status,
                             static_cast<cudaStream_t>(stream)),
         "launch");
  });
}

int ivc_kv_append(ivc_kv *h, const ivc_kv_cache *cache, const ivc_kv_seqs *seqs, int dtype, const ivc_rows *k,
                  const ivc_rows *v, const ivc_rotary *rotary, int q_heads, const ivc_rows *q, const ivc_rows *q_out,
                  void *stream) {
  return guarded(h, "ivc_kv_append", [&] {
    check_dtype(dtype);
    const ivb::KvCache c = check_cache(cache);
    const ivb::KvSeqs s = check_seqs(seqs);
    const ivb::KvRotary rot = rotation(rotary, c.dim, s.tokens);
    const ivb::KvRows kr = rows(k, "k is null", s.tokens, c.heads), vr = rows(v, "v is null", s.tokens, c.heads);
    need(q_heads >= 0 && q_heads <= 65536, "q_heads out of range");
    need(q_heads == 0 || rotary, "queries need a rotary");
    ivb::KvRows qr{}, qo{};
    if (q_heads) {
      qr = rows(q, "q is null", s.tokens, q_heads);
      qo = out_rows(q_out, "q_out is null", s.tokens, q_heads, c.dim);
    }
    if (s.tokens == 0) return;
    cuda(ivb::launch_kv_append(dtype == IVC_BF16, c, s, kr, vr, rot, q_heads, qr, qo, h->status,
                               static_cast<cudaStream_t>(stream)),
         "launch");
  });
}

int ivc_kv_read(ivc_kv *h, const ivc_kv_cache *cache, const ivc_kv_seqs *seqs, int dtype, const ivc_rows *k,
                const ivc_rows *v, void *stream) {
  return guarded(h, "ivc_kv_read", [&] {
    check_dtype(dtype);
    const ivb::KvCache c = check_cache(cache);
    const ivb::KvSeqs s = check_seqs(seqs);
    ivb::KvRows kr{}, vr{};
    if (k) kr = out_rows(k, "k is null", s.tokens, c.heads, c.dim);
    if (v) vr = out_rows(v, "v is null", s.tokens, c.heads, c.dim);
    if (s.tokens == 0 || (!k && !v)) return;
    cuda(ivb::launch_kv_read(dtype == IVC_BF16, c, s, kr, vr, h->status, static_cast<cudaStream_t>(stream)), "launch");
  });
}

int ivc_kv_attend(ivc_kv *h, const ivc_kv_cache *cache, const ivc_kv_seqs *seqs, int dtype, int q_heads, int max_new,
                  const ivc_rows *q, const ivc_rows *out, float scale, int window, int sinks, void *stream) {
  return guarded(h, "ivc_kv_attend", [&] {
    check_dtype(dtype);
    const ivb::KvAttend a = attention(h, cache, seqs, q_heads, max_new, q, out, scale, window, sinks);
    if (a.seqs.tokens == 0) return;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    cuda(ivb::launch_kv_attend(dtype == IVC_BF16, a, workspace(h, st), h->sms, st), "launch");
  });
}

int ivc_kv_attend_shared(ivc_kv *h, const ivc_kv_cache *cache, const ivc_kv_seqs *seqs, const ivc_kv_groups *groups,
                         int dtype, int q_heads, int max_new, const ivc_rows *q, const ivc_rows *out, float scale,
                         float *scratch, int64_t scratch_floats, void *stream) {
  return guarded(h, "ivc_kv_attend_shared", [&] {
    check_dtype(dtype);
    ivb::KvAttend a = attention(h, cache, seqs, q_heads, max_new, q, out, scale, 0, 0);
    need(groups != nullptr, "no groups");
    need(groups->count >= 0 && groups->count <= a.seqs.batch, "groups: at most one for each sequence");
    need(groups->count > 0 || a.seqs.batch == 0, "sequences without a group");
    need(groups->count == 0 || (groups->first && groups->shared), "the groups have a null pointer");
    need(aligned(groups->first, 4) && aligned(groups->shared, 4), "first and shared are int32");
    need(aligned(scratch, 16), "scratch is 16-byte aligned");
    need(a.seqs.tokens == 0 || (scratch && scratch_floats >= a.seqs.tokens * q_heads * (a.cache.dim + 2)),
         "scratch: at least tokens * q_heads * (head_dim + 2) floats");
    need(a.seqs.tokens * a.group < (1LL << 30), "tokens * q_heads / kv_heads out of range");
    if (a.seqs.tokens == 0) return;
    const Memory room(scratch, 4 * a.seqs.tokens * q_heads * (a.cache.dim + 2));
    const int64_t blocks = a.cache.pages * a.cache.heads * (a.cache.page / IVC_KV_BLOCK);
    need(!meet(a.q, a.seqs.tokens, q_heads, a.cache.dim, room) && !meet(a.out, a.seqs.tokens, q_heads, a.cache.dim, room),
         "scratch overlaps q or out");
    for (const void *p : {(const void *)a.cache.k, (const void *)a.cache.v})
      need(!meet(room, Memory(p, blocks * IVC_KV_BLOCK * a.cache.dim)), "scratch overlaps the cache");
    for (const void *p : {(const void *)a.cache.ks, (const void *)a.cache.vs}) need(!meet(room, Memory(p, 4 * blocks)), "scratch overlaps the cache");
    a.first = groups->first;
    a.shared = groups->shared;
    a.groups = groups->count;
    a.sequences = a.seqs.batch;
    a.scratch = scratch;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    cuda(ivb::launch_kv_attend_shared(dtype == IVC_BF16, a, workspace(h, st), h->sms, st), "launch");
  });
}

int ivc_kv_sample(ivc_kv *h, const ivc_logits *logits, const ivc_sampling *how, int32_t *tokens, float *probs,
                  void *stream) {
  return guarded(h, "ivc_kv_sample", [&] {
    need(logits && how, "null pointer");
    need(logits->dtype == IVC_F16 || logits->dtype == IVC_BF16 || logits->dtype == IVC_F32, "logits are IVC_F16, IVC_BF16 or IVC_F32");
    need(logits->rows >= 0 && logits->rows <= (1 << 24), "rows out of range");
    need(logits->vocab >= 1 && logits->vocab <= ivb::kSampleMaxVocab, "vocab: 1 to 500000");
    if (logits->rows == 0) return;
    need(logits->data && how->u && tokens, "null pointer");
    need(aligned(logits->data, logits->dtype == IVC_F32 ? 4 : 2), "logits are aligned to their type");
    need(aligned(how->u, 4) && aligned(how->temperature, 4) && aligned(how->top_k, 4) && aligned(how->top_p, 4) &&
             aligned(how->min_p, 4) && aligned(tokens, 4) && aligned(probs, 4),
         "the rows' numbers are 4-byte aligned");
    ivb::Sample s{};
    s.x = logits->data;
    s.rows = logits->rows;
    s.stride = logits->row_stride;
    s.vocab = (int)logits->vocab;
    s.dtype = logits->dtype;
    s.u = how->u, s.temperature = how->temperature, s.top_k = how->top_k, s.top_p = how->top_p, s.min_p = how->min_p;
    s.tokens = tokens;
    s.probs = probs;
    cuda(ivb::launch_sample(s, h->sms, static_cast<cudaStream_t>(stream)), "launch");
  });
}

int ivc_kv_mx4_quantize(ivc_kv *h, int dtype, const void *x, int64_t rows, int64_t x_stride, const ivc_mx4 *m,
                        void *stream) {
  return guarded(h, "ivc_kv_mx4_quantize", [&] {
    const ivb::Mx4 q = check_mx4(m);
    check_matrix(dtype, x, rows, q.width, x_stride, false);
    need(rows <= q.rows, "the 4-bit matrix has fewer rows");
    if (rows == 0) return;
    need(apart(matrix(x, rows, q.width, x_stride), first_rows(q, rows)), "the 4-bit matrix overlaps x");
    cuda(ivb::launch_mx4_quantize(dtype == IVC_BF16, x, rows, x_stride, q, h->sms, static_cast<cudaStream_t>(stream)), "launch");
  });
}

int ivc_kv_mx4_read(ivc_kv *h, const ivc_mx4 *m, int64_t rows, int dtype, void *out, int64_t out_stride, void *stream) {
  return guarded(h, "ivc_kv_mx4_read", [&] {
    const ivb::Mx4 q = check_mx4(m);
    check_matrix(dtype, out, rows, q.width, out_stride, true);
    need(rows <= q.rows, "the 4-bit matrix has fewer rows");
    if (rows == 0) return;
    need(apart(matrix(out, rows, q.width, out_stride), first_rows(q, rows)), "out overlaps the 4-bit matrix");
    cuda(ivb::launch_mx4_read(dtype == IVC_BF16, q, rows, out, out_stride, h->sms, static_cast<cudaStream_t>(stream)), "launch");
  });
}

int ivc_kv_mx4_linear(ivc_kv *h, int x_dtype, const void *x, int64_t rows, int64_t x_stride, const ivc_mx4 *xq,
                      const ivc_mx4 *w, int out_dtype, void *out, int64_t out_stride, void *stream) {
  return guarded(h, "ivc_kv_mx4_linear", [&] {
    ivb::Mx4Linear a{};
    a.x = check_mx4(xq);
    a.w = check_mx4(w);
    need(a.x.width == a.w.width, "the matrices differ in width");
    need(a.w.rows <= (1 << 26), "rows of the weights out of range");
    check_matrix(out_dtype, out, rows, a.w.rows, out_stride, true);
    if (x) check_matrix(x_dtype, x, rows, a.x.width, x_stride, false);
    need(rows <= a.x.rows, "the 4-bit matrix has fewer rows");
    if (rows == 0 || a.w.rows == 0) return;
    a.x.rows = rows;
    const Memory input = matrix(x, x ? rows : 0, a.x.width, x_stride), output = matrix(out, rows, a.w.rows, out_stride);
    need(!x || (apart(a.x, a.w) && apart(input, a.x)), "the room for x in 4 bits overlaps x or the weights");
    need(!meet(output, input) && apart(output, a.x) && apart(output, a.w), "out overlaps x, its room or the weights");
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    a.rows = x;
    a.x_stride = x_stride;
    a.x_bf16 = x_dtype == IVC_BF16;
    a.out = out;
    a.stride = out_stride;
    a.bf16 = out_dtype == IVC_BF16;
    a.status = h->status;
    a.sms = h->sms;
    a.device = h->device;
    cuda(ivb::launch_mx4_linear(a, st), "launch");
  });
}

}  // extern "C"
