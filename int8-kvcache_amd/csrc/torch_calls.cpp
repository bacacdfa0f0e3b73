// CPython calls into libkvq_int8.so for torch tensors: the operators' argument checks and the C ABI call in one
// native function, in place of ~40 attribute reads, ctypes conversions and formatted messages per call (18-30 us
// of host time, more than a decode-sized kernel takes).
//
// Each function returns 0 after the launch, the library's status if it refused the call, or DECLINED without
// having done anything when the arguments are not the plain form it knows (an exact torch.Tensor of dense GPU
// memory in every place, the documented shapes, layouts and dtypes). The caller then takes kvq.cuda_kernels'
// Python path, which repeats the checks, raises what is wrong or serves the form: nothing is accepted, refused
// or reported differently here. No C++ exception leaves a function.
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstdint>
#include <cstdlib>

#include "../../include/kvq_int8.h"

#ifndef KVQ_TORCH_VERSION
#error "KVQ_TORCH_VERSION: torch.__version__ of the headers in use (int8-kvcache_amd/build.py passes it)"
#endif
#define KVQ_TEXT_(x) #x
#define KVQ_TEXT(x) KVQ_TEXT_(x)

namespace {

constexpr long DECLINED = -1;

// What this file's calls were compiled against: the library's signatures, torch's tensor layout, the interpreter's
// objects. kvq._native binds the module only where all three are the running ones.
constexpr char BUILT_FOR[] = "abi " KVQ_TEXT(KVQ_ABI_VERSION) ", torch " KVQ_TORCH_VERSION ", python " KVQ_TEXT(
    PY_MAJOR_VERSION) "." KVQ_TEXT(PY_MINOR_VERSION);

// the library's entry points, by address (bind): whichever library file the package loaded
decltype(&kvq_quant_cache) p_quant_cache;
decltype(&kvq_int8_decode_attention) p_decode;
decltype(&kvq_int8_decode_attention_ex) p_decode_ex;
decltype(&kvq_dequant_pages) p_dequant;
decltype(&kvq_paged_prefill_attention_ex) p_prefill;
decltype(&kvq_int8_prefill_attention_ex) p_prefill_i8;
decltype(&kvq_quant_block_cache) p_quant_block;
decltype(&kvq_read_block_cache) p_read_block;
decltype(&kvq_block_decode_attention) p_block_decode;
decltype(&kvq_block_prefill_attention) p_block_prefill;
decltype(&kvq_block_codes) p_block_codes;
decltype(&kvq_quant_fp4_cache) p_quant_fp4;
decltype(&kvq_read_fp4_cache) p_read_fp4;
decltype(&kvq_fp4_pages) p_fp4_pages;
decltype(&kvq_fp4_prefill_attention) p_fp4_prefill;
decltype(&kvq_fp4_decode_attention) p_fp4_decode;
decltype(&kvq_fp4_key_weights) p_key_weights;
decltype(&kvq_fp4_evict) p_evict;
decltype(&kvq_norm_rope) p_norm_rope;

// A tensor argument this file may read: exactly torch.Tensor (or Parameter), dense GPU memory, no wrapper
// (functorch, functionalization, fake or subclass tensors go to the Python path).
const at::Tensor* tensor(PyObject* o) {
  if (!THPVariable_CheckExact(o)) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(o);
  if (!t.defined() || !t.is_cuda()) return nullptr;
  static const c10::DispatchKeySet plain({c10::DispatchKey::CUDA, c10::DispatchKey::AutogradCUDA,
                                          c10::DispatchKey::AutocastCUDA, c10::DispatchKey::ADInplaceOrView});
  if (!((t.key_set() | plain) == plain)) return nullptr;
  return &t;
}

bool as_int(PyObject* o, int64_t& v) {
  if (!PyLong_CheckExact(o)) return false;
  v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) {
    PyErr_Clear();
    return false;
  }
  return true;
}

// K / V scale tables: contiguous float32 [heads, 1 or d]; their columns, or 0
int64_t scale_cols(const at::Tensor& s, int64_t heads, int64_t d) {
  if (s.scalar_type() != at::kFloat || s.dim() != 2 || !s.is_contiguous() || s.size(0) != heads ||
      (s.size(1) != 1 && s.size(1) != d))
    return 0;
  return s.size(1);
}

template <typename... T>
bool one_device(const at::Tensor& first, const T&... rest) {
  return ((rest.device() == first.device()) && ...);
}

bool bf16_rows(const at::Tensor& t) { return t.dim() == 3 && t.scalar_type() == at::kBFloat16 && t.stride(2) == 1; }
bool int8_cache(const at::Tensor& k, const at::Tensor& v) {
  return k.dim() == 4 && v.dim() == 4 && k.scalar_type() == at::kChar && v.scalar_type() == at::kChar &&
         k.sizes() == v.sizes() && k.stride(3) == 1 && v.stride(3) == 1;
}
bool index_vector(const at::Tensor& t) { return t.dim() == 1 && t.scalar_type() == at::kInt && t.is_contiguous(); }

void* stream_of(const at::Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

// The entry point this thread's last call went to (its own record: the interpreter lock is not held meanwhile).
thread_local const char* entry = "";

// The C call with the interpreter lock released (as ctypes does): a full launch queue blocks this thread alone.
template <typename F>
long launch(const char* name, F&& f) {
  long rc;
  entry = name;
  Py_BEGIN_ALLOW_THREADS
  rc = f();
  Py_END_ALLOW_THREADS
  return rc;
}

template <typename F>
PyObject* guarded(F&& f) {
  long rc = DECLINED;
  try {
    rc = f();
  } catch (...) {
    rc = DECLINED;   // the Python path meets the same condition and reports it
  }
  return PyLong_FromLong(rc);
}

// (key, value, k_cache, v_cache, slots, k_scale, v_scale, k_mu)
PyObject* quant_cache(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> long {
    if (n != 8 || !p_quant_cache) return DECLINED;
    const at::Tensor* t[8];
    for (int i = 0; i < 8; ++i)
      if (!(t[i] = tensor(a[i]))) return DECLINED;
    const at::Tensor &key = *t[0], &value = *t[1], &kc = *t[2], &vc = *t[3], &slots = *t[4], &ks = *t[5], &vs = *t[6], &mu = *t[7];
    if (!bf16_rows(key) || !bf16_rows(value) || !int8_cache(kc, vc) || slots.dim() != 1 ||
        slots.scalar_type() != at::kLong || slots.stride(0) != 1 ||
        !one_device(key, value, kc, vc, slots, ks, vs, mu))
      return DECLINED;
    const int64_t T = slots.size(0), H = key.size(1), D = key.size(2);
    if (T == 0 || value.size(2) != D || kc.size(3) != D || kc.size(2) != H || key.size(0) < T || value.size(0) < T)
      return DECLINED;
    const int64_t kcols = scale_cols(ks, H, D), vcols = scale_cols(vs, H, D);
    if (!kcols || !vcols || mu.scalar_type() != at::kFloat || mu.dim() != 2 || !mu.is_contiguous() || mu.size(0) != H ||
        mu.size(1) != D)
      return DECLINED;
    void *kp = key.data_ptr(), *vp = value.data_ptr(), *st = stream_of(key);
    auto *kcp = (int8_t*)kc.data_ptr(), *vcp = (int8_t*)vc.data_ptr();
    auto* sp = (const int64_t*)slots.data_ptr();
    auto *ksp = (const float*)ks.data_ptr(), *vsp = (const float*)vs.data_ptr(), *mup = (const float*)mu.data_ptr();
    return launch("kvq_quant_cache", [&] {
      return p_quant_cache(kp, key.stride(0), key.stride(1), vp, value.stride(0), value.stride(1), kcp, kc.stride(0),
                           kc.stride(1), kc.stride(2), vcp, vc.stride(0), vc.stride(1), vc.stride(2), sp, T, H, D,
                           kc.size(0), kc.size(1), ksp, kcols, vsp, vcols, mup, st);
    });
  });
}

// (q, k_cache, v_cache, out, cu_seqlens_q, seq_lens, block_table, k_scale, v_scale, softmax_scale,
//  segm_out | None, segm_max | None, segm_sum | None, max_query_len, qmax, q_group | None, max_splits)
PyObject* decode_attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> long {
    if (n != 17 || !p_decode || !p_decode_ex || getenv("KVQ_TARGET_WAVES")) return DECLINED;
    const at::Tensor* t[9];
    for (int i = 0; i < 9; ++i)
      if (!(t[i] = tensor(a[i]))) return DECLINED;
    const at::Tensor &q = *t[0], &kc = *t[1], &vc = *t[2], &out = *t[3], &cu = *t[4], &sl = *t[5], &bt = *t[6], &ks = *t[7], &vs = *t[8];
    if (!PyFloat_CheckExact(a[9])) return DECLINED;
    const double scale = PyFloat_AS_DOUBLE(a[9]);
    int64_t maxq, qmax, max_splits, group = 0;
    if (!as_int(a[13], maxq) || !as_int(a[14], qmax) || !as_int(a[16], max_splits)) return DECLINED;
    if (!bf16_rows(q) || !bf16_rows(out) || !int8_cache(kc, vc) || !index_vector(cu) || !index_vector(sl) || bt.dim() != 2 ||
        bt.scalar_type() != at::kInt || bt.stride(1) != 1 || !one_device(q, kc, vc, out, cu, sl, bt, ks, vs))
      return DECLINED;
    const int64_t B = cu.size(0) - 1, T = q.size(0), Hq = q.size(1), D = q.size(2), bs = kc.size(1), Hkv = kc.size(2);
    if (B <= 0 || kc.size(3) != D || bs < 16 || (bs & (bs - 1)) || out.size(0) < T || out.size(1) != Hq || out.size(2) != D ||
        sl.size(0) < B || bt.size(0) < B || Hkv <= 0 || Hq % Hkv)
      return DECLINED;
    if (a[15] != Py_None && !as_int(a[15], group)) return DECLINED;
    if (a[15] == Py_None) group = D;
    if (group != D && group != 32) return DECLINED;
    const int64_t kcols = scale_cols(ks, Hkv, D), vcols = scale_cols(vs, Hkv, D);
    if (!kcols || !vcols) return DECLINED;
    int64_t S = 1, rows = 0, seg_st = 0, seg_sh = 0;
    float *sop = nullptr, *smp = nullptr, *ssp = nullptr;
    if (a[11] != Py_None) {
      const at::Tensor *so = tensor(a[10]), *sm = tensor(a[11]), *ss = tensor(a[12]);
      if (!so || !sm || !ss || so->dim() != 4 || sm->dim() != 3 || ss->dim() != 3 || !one_device(q, *so, *sm, *ss)) return DECLINED;
      S = sm->size(2);
      rows = sm->size(0);
      for (const at::Tensor* x : {so, sm, ss})
        if (x->scalar_type() != at::kFloat || x->size(0) != rows || x->size(1) != Hq || x->size(2) != S) return DECLINED;
      seg_st = sm->stride(0);
      seg_sh = sm->stride(1);
      if (S > max_splits || sm->stride(2) != 1 || ss->strides() != sm->strides() || so->size(3) != D || so->stride(3) != 1 ||
          so->stride(2) != D || so->stride(1) != seg_sh * D || so->stride(0) != seg_st * D)
        return DECLINED;
      sop = (float*)so->data_ptr();
      smp = (float*)sm->data_ptr();
      ssp = (float*)ss->data_ptr();
    } else if (a[10] != Py_None || a[12] != Py_None) {
      return DECLINED;
    }
    void *qp = q.data_ptr(), *op = out.data_ptr(), *st = stream_of(q);
    auto *kp = (const int8_t*)kc.data_ptr(), *vp = (const int8_t*)vc.data_ptr();
    auto *cup = (const int32_t*)cu.data_ptr(), *slp = (const int32_t*)sl.data_ptr(), *btp = (const int32_t*)bt.data_ptr();
    auto *ksp = (const float*)ks.data_ptr(), *vsp = (const float*)vs.data_ptr();
    const bool ex = group != D || rows < T;   // tokens past the buffers' rows are never cut
    return launch(ex ? "kvq_int8_decode_attention_ex" : "kvq_int8_decode_attention", [&] {
      if (ex)
        return p_decode_ex(qp, q.stride(0), q.stride(1), kp, kc.stride(0), kc.stride(1), kc.stride(2), vp, vc.stride(0),
                           vc.stride(1), vc.stride(2), kc.size(0), bs, Hkv, D, op, out.stride(0), out.stride(1), cup, slp,
                           btp, bt.stride(0), B, Hq, ksp, kcols, vsp, vcols, scale, sop, smp, ssp, seg_st, seg_sh, S, rows,
                           0, maxq, qmax, group, st);
      return p_decode(qp, q.stride(0), q.stride(1), kp, kc.stride(0), kc.stride(1), kc.stride(2), vp, vc.stride(0),
                      vc.stride(1), vc.stride(2), kc.size(0), bs, Hkv, D, op, out.stride(0), out.stride(1), cup, slp, btp,
                      bt.stride(0), B, Hq, ksp, kcols, vsp, vcols, scale, sop, smp, ssp, seg_st, seg_sh, S, 0, maxq, qmax,
                      st);
    });
  });
}

// (q, k_cache, v_cache, out, cu_seqlens_q, seq_lens, block_table, k_scale, v_scale, softmax_scale, mode,
//  rows_per_tile, tile_req, tile_row, tile_piece | None, tile_slot | None, merge | None, slots,
//  src_req, src_j, temporary block table)
// The long requests' attention with its scratch: mode 0 dequantizes their pages into a temporary bf16 cache and
// runs the bf16 prefill on it (the last three arguments), 1 and 2 read the INT8 pages (2: scales folded).
PyObject* long_attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> long {
    if (n != 21 || !p_dequant || !p_prefill || !p_prefill_i8) return DECLINED;
    const at::Tensor* t[9];
    for (int i = 0; i < 9; ++i)
      if (!(t[i] = tensor(a[i]))) return DECLINED;
    const at::Tensor &q = *t[0], &kc = *t[1], &vc = *t[2], &out = *t[3], &cu = *t[4], &sl = *t[5], &bt = *t[6], &ks = *t[7], &vs = *t[8];
    if (!PyFloat_CheckExact(a[9])) return DECLINED;
    const double scale = PyFloat_AS_DOUBLE(a[9]);
    int64_t mode, rows, slots;
    if (!as_int(a[10], mode) || !as_int(a[11], rows) || !as_int(a[17], slots) || mode < 0 || mode > 2) return DECLINED;
    const at::Tensor *treq = tensor(a[12]), *trow = tensor(a[13]);
    if (!treq || !trow || !index_vector(*treq) || !index_vector(*trow)) return DECLINED;
    const int64_t tiles = treq->size(0);
    if (!bf16_rows(q) || !bf16_rows(out) || !int8_cache(kc, vc) || cu.scalar_type() != at::kInt || sl.scalar_type() != at::kInt ||
        bt.dim() != 2 || bt.scalar_type() != at::kInt || bt.stride(1) != 1 || trow->size(0) != tiles || tiles == 0 ||
        !one_device(q, kc, vc, out, cu, sl, bt, ks, vs, *treq, *trow))
      return DECLINED;
    const int64_t Hq = q.size(1), D = q.size(2), nb = kc.size(0), bs = kc.size(1), H = kc.size(2);
    if (kc.size(3) != D || out.size(1) != Hq || out.size(2) != D || out.size(0) != q.size(0) || H <= 0) return DECLINED;
    const int64_t kcols = scale_cols(ks, H, D), vcols = scale_cols(vs, H, D);
    if (!kcols || !vcols) return DECLINED;
    const int32_t *pp = nullptr, *sp = nullptr, *mp = nullptr;
    int64_t nm = 0;
    at::Tensor part_out, part_ml;
    const auto f32 = q.options().dtype(at::kFloat);
    if (a[14] != Py_None) {
      const at::Tensor *piece = tensor(a[14]), *slot = tensor(a[15]), *merge = tensor(a[16]);
      if (!piece || !slot || !merge || !index_vector(*piece) || !index_vector(*slot) || piece->size(0) != tiles ||
          slot->size(0) != tiles || merge->scalar_type() != at::kInt || merge->dim() != 2 || !merge->is_contiguous() ||
          merge->size(1) != 4 || !one_device(q, *piece, *slot, *merge))
        return DECLINED;
      pp = (const int32_t*)piece->data_ptr();
      sp = (const int32_t*)slot->data_ptr();
      mp = (const int32_t*)merge->data_ptr();
      nm = merge->size(0);
      part_out = at::empty({slots, H, rows, D}, f32);
      part_ml = at::empty({slots, H, rows, 2}, f32);
    }
    float *pop = pp ? (float*)part_out.data_ptr() : nullptr, *pmp = pp ? (float*)part_ml.data_ptr() : nullptr;
    void *qp = q.data_ptr(), *op = out.data_ptr(), *st = stream_of(q);
    auto *kp = (const int8_t*)kc.data_ptr(), *vp = (const int8_t*)vc.data_ptr();
    auto *cup = (const int32_t*)cu.data_ptr(), *slp = (const int32_t*)sl.data_ptr(), *btp = (const int32_t*)bt.data_ptr();
    auto *ksp = (const float*)ks.data_ptr(), *vsp = (const float*)vs.data_ptr();
    auto *rp = (const int32_t*)treq->data_ptr(), *wp = (const int32_t*)trow->data_ptr();
    if (mode) {
      return launch(pp ? "kvq_int8_prefill_attention_ex" : "kvq_int8_prefill_attention", [&] {
        return p_prefill_i8(qp, q.stride(0), q.stride(1), kp, kc.stride(0), kc.stride(1), kc.stride(2), vp, vc.stride(0),
                            vc.stride(1), vc.stride(2), nb, bs, H, D, op, out.stride(0), out.stride(1), cup, slp, btp,
                            bt.stride(0), Hq, rp, wp, tiles, rows, scale, ksp, kcols, vsp, vcols, mode == 2, pp, sp, mp, nm,
                            pop, pmp, st);
      });
    }
    const at::Tensor *sreq = tensor(a[18]), *sj = tensor(a[19]), *tbt = tensor(a[20]);
    if (!sreq || !sj || !tbt || !index_vector(*sreq) || !index_vector(*sj) || sreq->size(0) == 0 ||
        sj->size(0) != sreq->size(0) || tbt->dim() != 2 || tbt->scalar_type() != at::kInt || tbt->stride(1) != 1 ||
        !one_device(q, *sreq, *sj, *tbt))
      return DECLINED;
    const int64_t P = sreq->size(0);
    const at::Tensor kt = at::empty({P, bs, H, D}, q.options()), vt = at::empty({P, bs, H, D}, q.options());
    void *ktp = kt.data_ptr(), *vtp = vt.data_ptr();
    auto *rqp = (const int32_t*)sreq->data_ptr(), *jp = (const int32_t*)sj->data_ptr(), *tbp = (const int32_t*)tbt->data_ptr();
    return launch("kvq_dequant_pages", [&] {
      const int rc = p_dequant(kp, kc.stride(0), kc.stride(1), kc.stride(2), vp, vc.stride(0), vc.stride(1), vc.stride(2), nb,
                               bs, H, D, ktp, vtp, btp, bt.stride(0), rqp, jp, P, ksp, kcols, vsp, vcols, st);
      if (rc) return rc;
      entry = pp ? "kvq_paged_prefill_attention_ex" : "kvq_paged_prefill_attention";
      return p_prefill(qp, q.stride(0), q.stride(1), ktp, bs * H * D, H * D, D, vtp, bs * H * D, H * D, D, P, bs, H, D, op,
                       out.stride(0), out.stride(1), cup, slp, tbp, tbt->stride(0), Hq, rp, wp, tiles, rows, scale, pp, sp, mp,
                       nm, pop, pmp, st);
    });
  });
}

// ---- block-scaled cache (kvq.block_cache) ----
// A cache's views and scales: int8 [nb, bs, H, D] and float32 [nb, H, blocks per page] of one layout.
struct BlockCache {
  const int8_t *k, *v;
  float *ks, *vs;
  int64_t kb, kn, kh, vb, vn, vh, nb, bs, H, D, sb, sh, sg, group;
  bool read(const at::Tensor& kc, const at::Tensor& vc, const at::Tensor& ks_t, const at::Tensor& vs_t) {
    if (!int8_cache(kc, vc) || ks_t.dim() != 3 || vs_t.dim() != 3 || ks_t.scalar_type() != at::kFloat ||
        vs_t.scalar_type() != at::kFloat || ks_t.sizes() != vs_t.sizes() || ks_t.strides() != vs_t.strides())
      return false;
    nb = kc.size(0), bs = kc.size(1), H = kc.size(2), D = kc.size(3);
    const int64_t blocks = ks_t.size(2);
    if (ks_t.size(0) != nb || ks_t.size(1) != H || blocks < 1 || bs % blocks) return false;
    group = bs / blocks;   // (the library refuses sizes it does not know)
    k = (const int8_t*)kc.data_ptr(), v = (const int8_t*)vc.data_ptr();
    ks = (float*)ks_t.data_ptr(), vs = (float*)vs_t.data_ptr();
    kb = kc.stride(0), kn = kc.stride(1), kh = kc.stride(2), vb = vc.stride(0), vn = vc.stride(1), vh = vc.stride(2);
    sb = ks_t.stride(0), sh = ks_t.stride(1), sg = ks_t.stride(2);
    return true;
  }
};
// the library sizes its grids for the current device: another one goes to the Python path, which switches
bool on_current(const at::Tensor& t) { return t.device().index() == c10::hip::current_device(); }
bool table(const at::Tensor& t, int64_t rows) {
  return t.dim() == 2 && t.scalar_type() == at::kInt && t.stride(1) == 1 && t.size(0) >= rows;
}

// (key, value, k_cache, v_cache, k_scale, v_scale, cu_seqlens_q, seq_lens, block_table)
PyObject* quant_block_cache(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> long {
    if (n != 9 || !p_quant_block) return DECLINED;
    const at::Tensor* t[9];
    for (int i = 0; i < 9; ++i)
      if (!(t[i] = tensor(a[i]))) return DECLINED;
    const at::Tensor &key = *t[0], &value = *t[1], &cu = *t[6], &sl = *t[7], &bt = *t[8];
    BlockCache c;
    if (!bf16_rows(key) || !bf16_rows(value) || !c.read(*t[2], *t[3], *t[4], *t[5]) || !index_vector(cu) || !index_vector(sl) ||
        !one_device(key, value, *t[2], *t[3], *t[4], *t[5], cu, sl, bt) || !on_current(key))
      return DECLINED;
    const int64_t T = key.size(0), B = cu.size(0) - 1;
    if (T == 0 || B <= 0 || key.sizes() != value.sizes() || key.size(1) != c.H || key.size(2) != c.D || sl.size(0) < B ||
        !table(bt, B))
      return DECLINED;
    void *kp = key.data_ptr(), *vp = value.data_ptr(), *st = stream_of(key);
    auto *cup = (const int32_t*)cu.data_ptr(), *slp = (const int32_t*)sl.data_ptr(), *btp = (const int32_t*)bt.data_ptr();
    return launch("kvq_quant_block_cache", [&] {
      return p_quant_block(kp, key.stride(0), key.stride(1), vp, value.stride(0), value.stride(1), T, (int8_t*)c.k, c.kb, c.kn,
                           c.kh, (int8_t*)c.v, c.vb, c.vn, c.vh, c.nb, c.bs, c.H, c.D, c.ks, c.vs, c.sb, c.sh, c.sg, c.group,
                           cup, slp, btp, bt.stride(0), B, st);
    });
  });
}

// (k_cache, v_cache, k_scale, v_scale, starts, cu_seqlens_k, block_table, k_out, v_out)
PyObject* read_block_cache(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> long {
    if (n != 9 || !p_read_block) return DECLINED;
    const at::Tensor* t[9];
    for (int i = 0; i < 9; ++i)
      if (!(t[i] = tensor(a[i]))) return DECLINED;
    const at::Tensor &start = *t[4], &cu = *t[5], &bt = *t[6], &ko = *t[7], &vo = *t[8];
    BlockCache c;
    if (!c.read(*t[0], *t[1], *t[2], *t[3]) || !index_vector(start) || !index_vector(cu) || !bf16_rows(ko) || !bf16_rows(vo) ||
        !one_device(ko, vo, *t[0], *t[1], *t[2], *t[3], start, cu, bt) || !on_current(ko))
      return DECLINED;
    const int64_t N = ko.size(0), B = cu.size(0) - 1;
    if (N == 0 || B <= 0 || ko.sizes() != vo.sizes() || ko.size(1) != c.H || ko.size(2) != c.D || start.size(0) < B ||
        !table(bt, B))
      return DECLINED;
    void *kp = ko.data_ptr(), *vp = vo.data_ptr(), *st = stream_of(ko);
    auto *sp = (const int32_t*)start.data_ptr(), *cup = (const int32_t*)cu.data_ptr(), *btp = (const int32_t*)bt.data_ptr();
    return launch("kvq_read_block_cache", [&] {
      return p_read_block(c.k, c.kb, c.kn, c.kh, c.v, c.vb, c.vn, c.vh, c.nb, c.bs, c.H, c.D, c.ks, c.vs, c.sb, c.sh, c.sg,
                          c.group, sp, cup, btp, bt.stride(0), B, kp, ko.stride(0), ko.stride(1), vp, vo.stride(0),
                          vo.stride(1), N, st);
    });
  });
}

// What both attention calls take: (q, k_cache, v_cache, out, cu_seqlens_q, seq_lens, block_table, k_scale, v_scale,
// softmax_scale, ...)
struct BlockAttn {
  BlockCache c;
  const at::Tensor *q, *out, *bt;
  const int32_t *cu, *sl;
  void *qp, *op, *st;
  int64_t B, T, Hq;
  double scale;
  bool read(PyObject* const* a) {
    const at::Tensor* t[9];
    for (int i = 0; i < 9; ++i)
      if (!(t[i] = tensor(a[i]))) return false;
    q = t[0], out = t[3], bt = t[6];
    if (!PyFloat_CheckExact(a[9])) return false;
    scale = PyFloat_AS_DOUBLE(a[9]);
    if (!bf16_rows(*q) || !bf16_rows(*out) || !c.read(*t[1], *t[2], *t[7], *t[8]) || !index_vector(*t[4]) ||
        !index_vector(*t[5]) || !one_device(*q, *t[1], *t[2], *out, *t[4], *t[5], *bt, *t[7], *t[8]) || !on_current(*q))
      return false;
    B = t[4]->size(0) - 1, T = q->size(0), Hq = q->size(1);
    if (B <= 0 || T == 0 || q->size(2) != c.D || out->size(0) < T || out->size(1) != Hq || out->size(2) != c.D ||
        t[5]->size(0) < B || !table(*bt, B) || c.H <= 0 || Hq % c.H)
      return false;
    cu = (const int32_t*)t[4]->data_ptr(), sl = (const int32_t*)t[5]->data_ptr();
    qp = q->data_ptr(), op = out->data_ptr(), st = stream_of(*q);
    return true;
  }
};

// (..., segm_out | None, segm_max | None, segm_sum | None, max_query_len, qmax, max_splits)
PyObject* block_decode_attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> long {
    if (n != 16 || !p_block_decode || getenv("KVQ_TARGET_WAVES")) return DECLINED;
    BlockAttn x;
    int64_t maxq, qmax, max_splits;
    if (!x.read(a) || !as_int(a[13], maxq) || !as_int(a[14], qmax) || !as_int(a[15], max_splits)) return DECLINED;
    int64_t S = 1, rows = 0, seg_st = 0, seg_sh = 0;
    float *sop = nullptr, *smp = nullptr, *ssp = nullptr;
    if (a[11] != Py_None) {
      const at::Tensor *so = tensor(a[10]), *sm = tensor(a[11]), *ss = tensor(a[12]);
      if (!so || !sm || !ss || so->dim() != 4 || sm->dim() != 3 || ss->dim() != 3 || !one_device(*x.q, *so, *sm, *ss))
        return DECLINED;
      S = sm->size(2), rows = sm->size(0), seg_st = sm->stride(0), seg_sh = sm->stride(1);
      for (const at::Tensor* y : {so, sm, ss})
        if (y->scalar_type() != at::kFloat || y->size(0) != rows || y->size(1) != x.Hq || y->size(2) != S) return DECLINED;
      const int64_t D = x.c.D;
      if (S > max_splits || sm->stride(2) != 1 || ss->strides() != sm->strides() || so->size(3) != D || so->stride(3) != 1 ||
          so->stride(2) != D || so->stride(1) != seg_sh * D || so->stride(0) != seg_st * D)
        return DECLINED;
      sop = (float*)so->data_ptr(), smp = (float*)sm->data_ptr(), ssp = (float*)ss->data_ptr();
    } else if (a[10] != Py_None || a[12] != Py_None) {
      return DECLINED;
    }
    const BlockCache& c = x.c;
    auto* btp = (const int32_t*)x.bt->data_ptr();
    return launch("kvq_block_decode_attention", [&] {
      return p_block_decode(x.qp, x.q->stride(0), x.q->stride(1), c.k, c.kb, c.kn, c.kh, c.v, c.vb, c.vn, c.vh, c.nb, c.bs, c.H,
                            c.D, c.ks, c.vs, c.sb, c.sh, c.sg, c.group, x.op, x.out->stride(0), x.out->stride(1), x.cu, x.sl,
                            btp, x.bt->stride(0), x.B, x.Hq, x.scale, sop, smp, ssp, seg_st, seg_sh, S, rows, 0, maxq, qmax,
                            x.st);
    });
  });
}

// (..., rows_per_tile, tile_req, tile_row, tile_piece | None, tile_slot | None, merge | None, slots,
//  src_req | None, src_j | None, temporary block table | None): the last three copy the pages' codes as bf16 first
PyObject* block_long_attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> long {
    if (n != 20 || !p_block_prefill || !p_block_codes) return DECLINED;
    BlockAttn x;
    int64_t rows, slots;
    if (!x.read(a) || !as_int(a[10], rows) || !as_int(a[16], slots)) return DECLINED;
    const at::Tensor *treq = tensor(a[11]), *trow = tensor(a[12]);
    if (!treq || !trow || !index_vector(*treq) || !index_vector(*trow) || !one_device(*x.q, *treq, *trow)) return DECLINED;
    const int64_t tiles = treq->size(0);
    if (tiles == 0 || trow->size(0) != tiles) return DECLINED;
    const int32_t *pp = nullptr, *sp = nullptr, *mp = nullptr;
    int64_t nm = 0;
    at::Tensor part_out, part_ml;
    if (a[13] != Py_None) {
      const at::Tensor *piece = tensor(a[13]), *slot = tensor(a[14]), *merge = tensor(a[15]);
      if (!piece || !slot || !merge || !index_vector(*piece) || !index_vector(*slot) || piece->size(0) != tiles ||
          slot->size(0) != tiles || merge->scalar_type() != at::kInt || merge->dim() != 2 || !merge->is_contiguous() ||
          merge->size(1) != 4 || !one_device(*x.q, *piece, *slot, *merge))
        return DECLINED;
      pp = (const int32_t*)piece->data_ptr(), sp = (const int32_t*)slot->data_ptr(), mp = (const int32_t*)merge->data_ptr();
      nm = merge->size(0);
      const auto f32 = x.q->options().dtype(at::kFloat);
      part_out = at::empty({slots, x.c.H, rows, x.c.D}, f32);
      part_ml = at::empty({slots, x.c.H, rows, 2}, f32);
    }
    float *pop = pp ? (float*)part_out.data_ptr() : nullptr, *pmp = pp ? (float*)part_ml.data_ptr() : nullptr;
    const BlockCache& c = x.c;
    auto* btp = (const int32_t*)x.bt->data_ptr();
    auto *rp = (const int32_t*)treq->data_ptr(), *wp = (const int32_t*)trow->data_ptr();
    const int32_t *rqp = nullptr, *jp = nullptr, *tbp = nullptr;
    int64_t P = 0, tbs = 0;
    at::Tensor kt, vt, st;
    if (a[17] != Py_None) {
      const at::Tensor *sreq = tensor(a[17]), *sj = tensor(a[18]), *tbt = tensor(a[19]);
      if (!sreq || !sj || !tbt || !index_vector(*sreq) || !index_vector(*sj) || sreq->size(0) == 0 ||
          sj->size(0) != sreq->size(0) || !table(*tbt, 0) || !one_device(*x.q, *sreq, *sj, *tbt))
        return DECLINED;
      P = sreq->size(0), tbs = tbt->stride(0);
      rqp = (const int32_t*)sreq->data_ptr(), jp = (const int32_t*)sj->data_ptr(), tbp = (const int32_t*)tbt->data_ptr();
      kt = at::empty({P, c.bs, c.H, c.D}, x.q->options());
      vt = at::empty({P, c.bs, c.H, c.D}, x.q->options());
      st = at::empty({c.H, P * (c.bs / 16), 4}, x.q->options().dtype(at::kFloat));
    }
    void *ktp = P ? kt.data_ptr() : nullptr, *vtp = P ? vt.data_ptr() : nullptr;
    float* stp = P ? (float*)st.data_ptr() : nullptr;
    return launch(P ? "kvq_block_codes" : "kvq_block_prefill_attention", [&] {
      if (P) {
        const int rc = p_block_codes(c.k, c.kb, c.kn, c.kh, c.v, c.vb, c.vn, c.vh, c.nb, c.bs, c.H, c.D, c.ks, c.vs, c.sb, c.sh,
                                     c.sg, c.group, ktp, vtp, stp, btp, x.bt->stride(0), rqp, jp, P, x.st);
        if (rc) return rc;
        entry = "kvq_block_prefill_attention";
      }
      return p_block_prefill(x.qp, x.q->stride(0), x.q->stride(1), c.k, c.kb, c.kn, c.kh, c.v, c.vb, c.vn, c.vh, c.nb, c.bs,
                             c.H, c.D, c.ks, c.vs, c.sb, c.sh, c.sg, c.group, x.op, x.out->stride(0), x.out->stride(1), x.cu,
                             x.sl, btp, x.bt->stride(0), x.Hq, rp, wp, tiles, rows, x.scale, pp, sp, mp, nm, pop, pmp, ktp,
                             vtp, stp, P, tbp, tbs, x.st);
    });
  });
}

// ---- 4-bit cache (kvq.fp4_cache) ----
// A cache's views and exponent bytes: uint8 [nb, bs, H, D / 2] and [nb, H, bs, D / 32].
struct Fp4Cache {
  uint8_t *k, *v, *ks, *vs;
  int64_t kb, kn, kh, vb, vn, vh, nb, bs, H, D, sb, sh;
  bool read(const at::Tensor& kc, const at::Tensor& vc, const at::Tensor& ks_t, const at::Tensor& vs_t) {
    if (kc.dim() != 4 || kc.scalar_type() != at::kByte || vc.scalar_type() != at::kByte || vc.sizes() != kc.sizes() ||
        kc.stride(3) != 1 || vc.stride(3) != 1)
      return false;
    nb = kc.size(0), bs = kc.size(1), H = kc.size(2), D = 2 * kc.size(3);
    if (bs < 16 || (bs & (bs - 1))) return false;
    for (const at::Tensor* s : {&ks_t, &vs_t})
      if (s->dim() != 4 || s->scalar_type() != at::kByte || s->size(0) != nb || s->size(1) != H || s->size(2) != bs ||
          s->size(3) != D / 32 || s->stride(3) != 1 || s->stride(2) != D / 32 || s->strides() != ks_t.strides())
        return false;
    k = (uint8_t*)kc.data_ptr(), v = (uint8_t*)vc.data_ptr(), ks = (uint8_t*)ks_t.data_ptr(), vs = (uint8_t*)vs_t.data_ptr();
    kb = kc.stride(0), kn = kc.stride(1), kh = kc.stride(2), vb = vc.stride(0), vn = vc.stride(1), vh = vc.stride(2);
    sb = ks_t.stride(0), sh = ks_t.stride(1);
    return true;
  }
};
bool bf16_rows_of(const at::Tensor& t, int64_t heads, int64_t d) { return bf16_rows(t) && t.size(1) == heads && t.size(2) == d; }
bool lse_rows(const at::Tensor& t, int64_t rows, int64_t heads) {
  return t.dim() == 2 && t.scalar_type() == at::kFloat && t.stride(1) == 1 && t.size(0) >= rows && t.size(1) == heads;
}

// (key, value, k_cache, v_cache, k_scale, v_scale, slot_mapping)
PyObject* quant_fp4_cache(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> long {
    if (n != 7 || !p_quant_fp4) return DECLINED;
    const at::Tensor* t[7];
    for (int i = 0; i < 7; ++i)
      if (!(t[i] = tensor(a[i]))) return DECLINED;
    const at::Tensor &key = *t[0], &value = *t[1], &slots = *t[6];
    Fp4Cache c;
    if (!c.read(*t[2], *t[3], *t[4], *t[5]) || !bf16_rows_of(key, c.H, c.D) || !bf16_rows(value) || key.sizes() != value.sizes() ||
        slots.dim() != 1 || slots.scalar_type() != at::kLong || slots.stride(0) != 1 || slots.size(0) == 0 ||
        slots.size(0) > key.size(0) || !one_device(key, value, *t[2], *t[3], *t[4], *t[5], slots) || !on_current(key))
      return DECLINED;
    const int64_t T = slots.size(0);
    void *kp = key.data_ptr(), *vp = value.data_ptr(), *st = stream_of(key);
    auto* sp = (const int64_t*)slots.data_ptr();
    return launch("kvq_quant_fp4_cache", [&] {
      return p_quant_fp4(kp, key.stride(0), key.stride(1), vp, value.stride(0), value.stride(1), c.k, c.kb, c.kn, c.kh, c.v, c.vb,
                         c.vn, c.vh, c.nb, c.bs, c.H, c.D, c.ks, c.vs, c.sb, c.sh, sp, T, st);
    });
  });
}

// (k_cache, v_cache, k_scale, v_scale, starts, cu_seqlens_k, block_table, k_out, v_out)
PyObject* read_fp4_cache(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> long {
    if (n != 9 || !p_read_fp4) return DECLINED;
    const at::Tensor* t[9];
    for (int i = 0; i < 9; ++i)
      if (!(t[i] = tensor(a[i]))) return DECLINED;
    const at::Tensor &start = *t[4], &cu = *t[5], &bt = *t[6], &ko = *t[7], &vo = *t[8];
    Fp4Cache c;
    if (!c.read(*t[0], *t[1], *t[2], *t[3]) || !index_vector(start) || !index_vector(cu) || !bf16_rows_of(ko, c.H, c.D) ||
        !bf16_rows(vo) || ko.sizes() != vo.sizes() || !one_device(ko, vo, *t[0], *t[1], *t[2], *t[3], start, cu, bt) ||
        !on_current(ko))
      return DECLINED;
    const int64_t N = ko.size(0), B = cu.size(0) - 1;
    if (N == 0 || B <= 0 || start.size(0) < B || !table(bt, B)) return DECLINED;
    void *kp = ko.data_ptr(), *vp = vo.data_ptr(), *st = stream_of(ko);
    auto *sp = (const int32_t*)start.data_ptr(), *cup = (const int32_t*)cu.data_ptr(), *btp = (const int32_t*)bt.data_ptr();
    return launch("kvq_read_fp4_cache", [&] {
      return p_read_fp4(c.k, c.kb, c.kn, c.kh, c.v, c.vb, c.vn, c.vh, c.nb, c.bs, c.H, c.D, c.ks, c.vs, c.sb, c.sh, sp, cup, btp,
                        bt.stride(0), B, kp, ko.stride(0), ko.stride(1), vp, vo.stride(0), vo.stride(1), N, st);
    });
  });
}

// What both attention calls take: (q, k_cache, v_cache, out, cu_seqlens_q, seq_lens, block_table, k_scale, v_scale,
// softmax_scale, ...)
struct Fp4Attn {
  Fp4Cache c;
  const at::Tensor *q, *out, *bt;
  const int32_t *cu, *sl;
  void *qp, *op, *st;
  int64_t B, T, Hq;
  double scale;
  bool read(PyObject* const* a) {
    const at::Tensor* t[9];
    for (int i = 0; i < 9; ++i)
      if (!(t[i] = tensor(a[i]))) return false;
    q = t[0], out = t[3], bt = t[6];
    if (!PyFloat_CheckExact(a[9])) return false;
    scale = PyFloat_AS_DOUBLE(a[9]);
    if (!bf16_rows(*q) || !c.read(*t[1], *t[2], *t[7], *t[8]) || !index_vector(*t[4]) || !index_vector(*t[5]) ||
        !one_device(*q, *t[1], *t[2], *out, *t[4], *t[5], *bt, *t[7], *t[8]) || !on_current(*q))
      return false;
    B = t[4]->size(0) - 1, T = q->size(0), Hq = q->size(1);
    if (B <= 0 || T == 0 || q->size(2) != c.D || !bf16_rows_of(*out, Hq, c.D) || out->size(0) < T || t[5]->size(0) < B ||
        !table(*bt, B) || c.H <= 0 || Hq % c.H)
      return false;
    cu = (const int32_t*)t[4]->data_ptr(), sl = (const int32_t*)t[5]->data_ptr();
    qp = q->data_ptr(), op = out->data_ptr(), st = stream_of(*q);
    return true;
  }
};

// (..., segm_out | None, segm_max | None, segm_sum | None, max_query_len, qmax, max_splits, lse | None)
PyObject* fp4_decode_attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> long {
    if (n != 17 || !p_fp4_decode || getenv("KVQ_TARGET_WAVES")) return DECLINED;
    Fp4Attn x;
    int64_t maxq, qmax, max_splits;
    if (!x.read(a) || !as_int(a[13], maxq) || !as_int(a[14], qmax) || !as_int(a[15], max_splits)) return DECLINED;
    int64_t S = 1, rows = 0, seg_st = 0, seg_sh = 0, lse_st = 0;
    float *sop = nullptr, *smp = nullptr, *ssp = nullptr, *lp = nullptr;
    if (a[11] != Py_None) {
      const at::Tensor *so = tensor(a[10]), *sm = tensor(a[11]), *ss = tensor(a[12]);
      if (!so || !sm || !ss || so->dim() != 4 || sm->dim() != 3 || ss->dim() != 3 || !one_device(*x.q, *so, *sm, *ss))
        return DECLINED;
      S = sm->size(2), rows = sm->size(0), seg_st = sm->stride(0), seg_sh = sm->stride(1);
      for (const at::Tensor* y : {so, sm, ss})
        if (y->scalar_type() != at::kFloat || y->size(0) != rows || y->size(1) != x.Hq || y->size(2) != S) return DECLINED;
      const int64_t D = x.c.D;
      if (S > max_splits || sm->stride(2) != 1 || ss->strides() != sm->strides() || so->size(3) != D || so->stride(3) != 1 ||
          so->stride(2) != D || so->stride(1) != seg_sh * D || so->stride(0) != seg_st * D)
        return DECLINED;
      sop = (float*)so->data_ptr(), smp = (float*)sm->data_ptr(), ssp = (float*)ss->data_ptr();
    } else if (a[10] != Py_None || a[12] != Py_None) {
      return DECLINED;
    }
    if (a[16] != Py_None) {
      const at::Tensor* lse = tensor(a[16]);
      if (!lse || !lse_rows(*lse, x.T, x.Hq) || !one_device(*x.q, *lse)) return DECLINED;
      lp = (float*)lse->data_ptr(), lse_st = lse->stride(0);
    }
    const Fp4Cache& c = x.c;
    auto* btp = (const int32_t*)x.bt->data_ptr();
    return launch("kvq_fp4_decode_attention", [&] {
      return p_fp4_decode(x.qp, x.q->stride(0), x.q->stride(1), c.k, c.kb, c.kn, c.kh, c.v, c.vb, c.vn, c.vh, c.nb, c.bs, c.H, c.D,
                          c.ks, c.vs, c.sb, c.sh, x.op, x.out->stride(0), x.out->stride(1), x.cu, x.sl, btp, x.bt->stride(0), x.B,
                          x.Hq, x.scale, sop, smp, ssp, seg_st, seg_sh, S, rows, lp, lse_st, 0, maxq, qmax, x.st);
    });
  });
}

// (..., rows_per_tile, tile_req, tile_row, tile_piece | None, tile_slot | None, merge | None, slots, src_req, src_j,
//  temporary block table)
PyObject* fp4_long_attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> long {
    if (n != 20 || !p_fp4_pages || !p_fp4_prefill) return DECLINED;
    Fp4Attn x;
    int64_t rows, slots;
    if (!x.read(a) || !as_int(a[10], rows) || !as_int(a[16], slots)) return DECLINED;
    const at::Tensor *treq = tensor(a[11]), *trow = tensor(a[12]);
    if (!treq || !trow || !index_vector(*treq) || !index_vector(*trow) || !one_device(*x.q, *treq, *trow)) return DECLINED;
    const int64_t tiles = treq->size(0);
    if (tiles == 0 || trow->size(0) != tiles) return DECLINED;
    const int32_t *pp = nullptr, *sp = nullptr, *mp = nullptr;
    int64_t nm = 0;
    at::Tensor part_out, part_ml;
    if (a[13] != Py_None) {
      const at::Tensor *piece = tensor(a[13]), *slot = tensor(a[14]), *merge = tensor(a[15]);
      if (!piece || !slot || !merge || !index_vector(*piece) || !index_vector(*slot) || piece->size(0) != tiles ||
          slot->size(0) != tiles || merge->scalar_type() != at::kInt || merge->dim() != 2 || !merge->is_contiguous() ||
          merge->size(1) != 4 || !one_device(*x.q, *piece, *slot, *merge))
        return DECLINED;
      pp = (const int32_t*)piece->data_ptr(), sp = (const int32_t*)slot->data_ptr(), mp = (const int32_t*)merge->data_ptr();
      nm = merge->size(0);
      const auto f32 = x.q->options().dtype(at::kFloat);
      part_out = at::empty({slots, x.c.H, rows, x.c.D}, f32);
      part_ml = at::empty({slots, x.c.H, rows, 2}, f32);
    }
    float *pop = pp ? (float*)part_out.data_ptr() : nullptr, *pmp = pp ? (float*)part_ml.data_ptr() : nullptr;
    const Fp4Cache& c = x.c;
    auto* btp = (const int32_t*)x.bt->data_ptr();
    auto *rp = (const int32_t*)treq->data_ptr(), *wp = (const int32_t*)trow->data_ptr();
    const at::Tensor *sreq = tensor(a[17]), *sj = tensor(a[18]), *tbt = tensor(a[19]);
    if (!sreq || !sj || !tbt || !index_vector(*sreq) || !index_vector(*sj) || sreq->size(0) == 0 ||
        sj->size(0) != sreq->size(0) || !table(*tbt, 0) || !one_device(*x.q, *sreq, *sj, *tbt))
      return DECLINED;
    const int64_t P = sreq->size(0), tbs = tbt->stride(0);
    auto *rqp = (const int32_t*)sreq->data_ptr(), *jp = (const int32_t*)sj->data_ptr(), *tbp = (const int32_t*)tbt->data_ptr();
    const at::Tensor kt = at::empty({P, c.bs, c.H, c.D}, x.q->options()), vt = at::empty({P, c.bs, c.H, c.D}, x.q->options());
    const at::Tensor st = at::empty({c.H, P * (c.bs / 16), 4}, x.q->options().dtype(at::kFloat));
    void *ktp = kt.data_ptr(), *vtp = vt.data_ptr();
    auto* stp = (float*)st.data_ptr();
    return launch("kvq_fp4_pages", [&] {
      const int rc = p_fp4_pages(c.k, c.kb, c.kn, c.kh, c.v, c.vb, c.vn, c.vh, c.nb, c.bs, c.H, c.D, c.ks, c.vs, c.sb, c.sh, ktp,
                                 vtp, stp, btp, x.bt->stride(0), rqp, jp, P, x.st);
      if (rc) return rc;
      entry = "kvq_fp4_prefill_attention";
      return p_fp4_prefill(x.qp, x.q->stride(0), x.q->stride(1), ktp, vtp, stp, P, c.bs, c.H, c.D, x.op, x.out->stride(0),
                           x.out->stride(1), x.cu, x.sl, tbp, tbs, x.Hq, rp, wp, tiles, rows, x.scale, pp, sp, mp, nm, pop, pmp,
                           x.st);
    });
  });
}

// (q, k_cache, k_scale, lse, weights, cu_seqlens_q, seq_lens, block_table, softmax_scale, max_query_len, qmax)
PyObject* add_key_weights(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> long {
    if (n != 11 || !p_key_weights) return DECLINED;
    const at::Tensor* t[8];
    for (int i = 0; i < 8; ++i)
      if (!(t[i] = tensor(a[i]))) return DECLINED;
    const at::Tensor &q = *t[0], &kc = *t[1], &ks = *t[2], &lse = *t[3], &w = *t[4], &cu = *t[5], &sl = *t[6], &bt = *t[7];
    if (!PyFloat_CheckExact(a[8])) return DECLINED;
    const double scale = PyFloat_AS_DOUBLE(a[8]);
    int64_t maxq, qmax;
    Fp4Cache c;
    if (!as_int(a[9], maxq) || !as_int(a[10], qmax) || !c.read(kc, kc, ks, ks) || !bf16_rows(q) || !index_vector(cu) ||
        !index_vector(sl) || !one_device(q, kc, ks, lse, w, cu, sl, bt) || !on_current(q))
      return DECLINED;
    const int64_t B = cu.size(0) - 1, T = q.size(0), Hq = q.size(1);
    if (B <= 0 || T == 0 || q.size(2) != c.D || c.H <= 0 || Hq % c.H || sl.size(0) < B || !table(bt, B) || !lse_rows(lse, T, Hq) ||
        w.dim() != 3 || w.scalar_type() != at::kFloat || w.stride(2) != 1 || w.size(0) < B || w.size(1) != c.H || w.size(2) == 0)
      return DECLINED;
    void *qp = q.data_ptr(), *st = stream_of(q);
    auto* lp = (const float*)lse.data_ptr();
    auto* wp = (float*)w.data_ptr();
    auto *cup = (const int32_t*)cu.data_ptr(), *slp = (const int32_t*)sl.data_ptr(), *btp = (const int32_t*)bt.data_ptr();
    return launch("kvq_fp4_key_weights", [&] {
      return p_key_weights(qp, q.stride(0), q.stride(1), c.k, c.kb, c.kn, c.kh, c.nb, c.bs, c.H, c.D, c.ks, c.sb, c.sh, lp,
                           lse.stride(0), wp, w.stride(0), w.stride(1), w.size(2), cup, slp, btp, bt.stride(0), B, Hq, scale, maxq,
                           qmax, st);
    });
  });
}

// (k_cache, v_cache, k_scale, v_scale, weights, seq_lens, keep, recent, block_table, kept, new_lens)
PyObject* evict_keys(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> long {
    if (n != 11 || !p_evict) return DECLINED;
    const at::Tensor* t[11];
    for (int i = 0; i < 11; ++i)
      if (i != 7 && !(t[i] = tensor(a[i]))) return DECLINED;
    const at::Tensor &kc = *t[0], &vc = *t[1], &w = *t[4], &sl = *t[5], &keep = *t[6], &bt = *t[8], &kept = *t[9], &nl = *t[10];
    int64_t recent;
    Fp4Cache c;
    if (!as_int(a[7], recent) || recent < 0 || !c.read(kc, vc, *t[2], *t[3]) || !index_vector(sl) || !index_vector(keep) ||
        !index_vector(nl) || !one_device(kc, vc, *t[2], *t[3], w, sl, keep, bt, kept, nl) || !on_current(kc))
      return DECLINED;
    const int64_t B = sl.size(0);
    if (B == 0 || keep.size(0) < B || nl.size(0) < B || !table(bt, B) || w.dim() != 3 || w.scalar_type() != at::kFloat ||
        w.stride(2) != 1 || w.size(0) < B || w.size(1) != c.H || kept.dim() != 3 || kept.scalar_type() != at::kInt ||
        kept.stride(2) != 1 || kept.size(0) < B || kept.size(1) != c.H)
      return DECLINED;
    void* st = stream_of(kc);
    auto* wp = (float*)w.data_ptr();
    auto *slp = (const int32_t*)sl.data_ptr(), *kp = (const int32_t*)keep.data_ptr(), *btp = (const int32_t*)bt.data_ptr();
    auto *op = (int32_t*)kept.data_ptr(), *np = (int32_t*)nl.data_ptr();
    return launch("kvq_fp4_evict", [&] {
      return p_evict(c.k, c.kb, c.kn, c.kh, c.v, c.vb, c.vn, c.vh, c.nb, c.bs, c.H, c.D, c.ks, c.vs, c.sb, c.sh, wp, w.stride(0),
                     w.stride(1), w.size(2), slp, kp, recent, btp, bt.stride(0), bt.size(1), B, op, kept.stride(0), kept.stride(1),
                     kept.size(2), np, st);
    });
  });
}

// (q, k, positions, cos_sin, q_weight | None, k_weight | None, eps, interleaved, q_out, k_out)
PyObject* norm_rope(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> long {
    if (n != 10 || !p_norm_rope || !PyFloat_CheckExact(a[6]) || !PyBool_Check(a[7])) return DECLINED;
    const at::Tensor *qt = tensor(a[0]), *kt = tensor(a[1]), *pt = tensor(a[2]), *tt = tensor(a[3]), *qot = tensor(a[8]),
                     *kot = tensor(a[9]);
    if (!qt || !kt || !pt || !tt || !qot || !kot) return DECLINED;
    const at::Tensor &q = *qt, &k = *kt, &pos = *pt, &tab = *tt, &qo = *qot, &ko = *kot;
    if (!bf16_rows(q) || !bf16_rows(k) || !bf16_rows(qo) || !bf16_rows(ko) || qo.sizes() != q.sizes() || ko.sizes() != k.sizes() ||
        k.size(0) != q.size(0) || k.size(2) != q.size(2) || q.size(0) == 0 || pos.dim() != 1 || pos.size(0) != q.size(0) ||
        (pos.scalar_type() != at::kInt && pos.scalar_type() != at::kLong) || !pos.is_contiguous() || tab.dim() != 2 ||
        (tab.scalar_type() != at::kFloat && tab.scalar_type() != at::kBFloat16) || tab.stride(1) != 1 ||
        !one_device(q, k, pos, tab, qo, ko) || !on_current(q))
      return DECLINED;
    const void *qw = nullptr, *kw = nullptr;
    bool wide = false;
    if (a[4] != Py_None || a[5] != Py_None) {
      const at::Tensor *x = tensor(a[4]), *y = tensor(a[5]);
      if (!x || !y || x->dim() != 1 || x->size(0) != q.size(2) || x->sizes() != y->sizes() || x->scalar_type() != y->scalar_type() ||
          (x->scalar_type() != at::kFloat && x->scalar_type() != at::kBFloat16) || !x->is_contiguous() || !y->is_contiguous() ||
          !one_device(q, *x, *y))
        return DECLINED;
      qw = x->data_ptr(), kw = y->data_ptr(), wide = x->scalar_type() == at::kFloat;
    }
    const double eps = PyFloat_AS_DOUBLE(a[6]);
    const bool inter = a[7] == Py_True;
    void *qp = q.data_ptr(), *kp = k.data_ptr(), *qop = qo.data_ptr(), *kop = ko.data_ptr(), *st = stream_of(q);
    const void *pp = pos.data_ptr(), *tp = tab.data_ptr();
    return launch("kvq_norm_rope", [&] {
      return p_norm_rope(qp, q.stride(0), q.stride(1), kp, k.stride(0), k.stride(1), qop, qo.stride(0), qo.stride(1), kop,
                         ko.stride(0), ko.stride(1), q.size(0), q.size(1), k.size(1), q.size(2), pp,
                         pos.scalar_type() == at::kLong ? 64 : 32, tp, tab.stride(0), tab.size(0), tab.size(1),
                         tab.scalar_type() == at::kBFloat16, qw, kw, !wide, eps, inter, st);
    });
  });
}

// (): the entry point of this thread's last call, as the Python path names it in its error
PyObject* last_entry(PyObject*, PyObject*) { return PyUnicode_FromString(entry); }

// ({name: address}): the library's entry points
PyObject* bind(PyObject*, PyObject* d) {
  auto at_name = [&](const char* nm) -> void* {
    PyObject* v = PyDict_Check(d) ? PyDict_GetItemString(d, nm) : nullptr;
    return v ? PyLong_AsVoidPtr(v) : nullptr;
  };
  p_quant_cache = (decltype(p_quant_cache))at_name("kvq_quant_cache");
  p_decode = (decltype(p_decode))at_name("kvq_int8_decode_attention");
  p_decode_ex = (decltype(p_decode_ex))at_name("kvq_int8_decode_attention_ex");
  p_dequant = (decltype(p_dequant))at_name("kvq_dequant_pages");
  p_prefill = (decltype(p_prefill))at_name("kvq_paged_prefill_attention_ex");
  p_prefill_i8 = (decltype(p_prefill_i8))at_name("kvq_int8_prefill_attention_ex");
  p_quant_block = (decltype(p_quant_block))at_name("kvq_quant_block_cache");
  p_read_block = (decltype(p_read_block))at_name("kvq_read_block_cache");
  p_block_decode = (decltype(p_block_decode))at_name("kvq_block_decode_attention");
  p_block_prefill = (decltype(p_block_prefill))at_name("kvq_block_prefill_attention");
  p_block_codes = (decltype(p_block_codes))at_name("kvq_block_codes");
  p_quant_fp4 = (decltype(p_quant_fp4))at_name("kvq_quant_fp4_cache");
  p_read_fp4 = (decltype(p_read_fp4))at_name("kvq_read_fp4_cache");
  p_fp4_pages = (decltype(p_fp4_pages))at_name("kvq_fp4_pages");
  p_fp4_prefill = (decltype(p_fp4_prefill))at_name("kvq_fp4_prefill_attention");
  p_fp4_decode = (decltype(p_fp4_decode))at_name("kvq_fp4_decode_attention");
  p_key_weights = (decltype(p_key_weights))at_name("kvq_fp4_key_weights");
  p_evict = (decltype(p_evict))at_name("kvq_fp4_evict");
  p_norm_rope = (decltype(p_norm_rope))at_name("kvq_norm_rope");
  if (PyErr_Occurred()) return nullptr;
  Py_RETURN_NONE;
}

PyMethodDef methods[] = {
    {"bind", bind, METH_O, "bind({entry point: address})"},
    {"quant_cache", (PyCFunction)(void (*)(void))quant_cache, METH_FASTCALL, "kvq_quant_cache on torch tensors"},
    {"decode_attention", (PyCFunction)(void (*)(void))decode_attention, METH_FASTCALL,
     "kvq_int8_decode_attention on torch tensors"},
    {"long_attention", (PyCFunction)(void (*)(void))long_attention, METH_FASTCALL,
     "the long requests' attention on torch tensors"},
    {"quant_block_cache", (PyCFunction)(void (*)(void))quant_block_cache, METH_FASTCALL,
     "kvq_quant_block_cache on torch tensors"},
    {"read_block_cache", (PyCFunction)(void (*)(void))read_block_cache, METH_FASTCALL,
     "kvq_read_block_cache on torch tensors"},
    {"block_decode_attention", (PyCFunction)(void (*)(void))block_decode_attention, METH_FASTCALL,
     "kvq_block_decode_attention on torch tensors"},
    {"block_long_attention", (PyCFunction)(void (*)(void))block_long_attention, METH_FASTCALL,
     "kvq_block_prefill_attention on torch tensors"},
    {"quant_fp4_cache", (PyCFunction)(void (*)(void))quant_fp4_cache, METH_FASTCALL,
     "kvq_quant_fp4_cache on torch tensors"},
    {"read_fp4_cache", (PyCFunction)(void (*)(void))read_fp4_cache, METH_FASTCALL,
     "kvq_read_fp4_cache on torch tensors"},
    {"fp4_decode_attention", (PyCFunction)(void (*)(void))fp4_decode_attention, METH_FASTCALL,
     "kvq_fp4_decode_attention on torch tensors"},
    {"fp4_long_attention", (PyCFunction)(void (*)(void))fp4_long_attention, METH_FASTCALL,
     "the long requests' attention over a 4-bit cache on torch tensors"},
    {"add_key_weights", (PyCFunction)(void (*)(void))add_key_weights, METH_FASTCALL,
     "kvq_fp4_key_weights on torch tensors"},
    {"evict_keys", (PyCFunction)(void (*)(void))evict_keys, METH_FASTCALL,
     "kvq_fp4_evict on torch tensors"},
    {"norm_rope", (PyCFunction)(void (*)(void))norm_rope, METH_FASTCALL,
     "kvq_norm_rope on torch tensors"},
    {"last_entry", last_entry, METH_NOARGS, "the entry point of this thread's last call"},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_torch_calls", "kvq operators on torch tensors", -1, methods, nullptr, nullptr,
                      nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__torch_calls(void) {
  PyObject* m = PyModule_Create(&module);
  if (m) PyModule_AddIntConstant(m, "DECLINED", DECLINED);
  if (m) PyModule_AddStringConstant(m, "BUILT_FOR", BUILT_FOR);
  return m;
}
