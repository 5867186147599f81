"""exactinfer forward pass on B200 (sm_100a): Python host side over the C ABI of libelb.so.

`Weight` and the free functions mirror the reference's operator interface (src/ops.h:11-29: matvec, get_row, rmsnorm);
`Backend` mirrors el::Backend (src/model.h:42-51: cfg, n_ctx, name, eval). All arithmetic runs in the CUDA library.
"""
from __future__ import annotations

import ctypes as C
import operator
import os

import numpy as np

from . import capi, synth
from .capi import Config, ElbError, check, lib

__all__ = ["Weight", "Backend", "Rope", "KvCache", "KvBatch", "beam_select", "beam_select_work", "cuda_available", "matvec", "get_row", "rmsnorm", "split_limbs", "synth", "Config",
           "ElbError"]


def cuda_available():
    """el::cuda_available (src/model.h:56): (ok, why)"""
    n = lib().elb_device_count()
    return (True, "") if n > 0 else (False, lib().elb_last_error().decode(errors="replace"))


class DeviceBuffer:
    def __init__(self, nbytes: int, device: int = 0):
        p = C.c_void_p()
        check(lib().elb_malloc(device, nbytes, C.byref(p)))
        self.ptr, self.nbytes = p, nbytes

    @classmethod
    def from_array(cls, a: np.ndarray, device: int = 0):
        a = np.ascontiguousarray(a)
        b = cls(a.nbytes, device)
        check(lib().elb_memcpy_h2d(b.ptr, a.ctypes.data_as(C.c_void_p), a.nbytes))
        return b

    def to_array(self, dtype, shape):
        out = np.empty(shape, dtype=dtype)
        check(lib().elb_memcpy_d2h(out.ctypes.data_as(C.c_void_p), self.ptr, out.nbytes))
        return out

    def free(self):
        if self.ptr:
            lib().elb_free(self.ptr)
            self.ptr = None

    def __del__(self):
        self.free()


class Weight:
    """One weight matrix in a ggml block format on the device (el::Tensor + upload_group of the reference)."""

    def __init__(self, ggml_type: int, rows: int, n: int, data: np.ndarray, planes: bool = False, pair: bool = False,
                 device: int = 0):
        data = np.ascontiguousarray(data, dtype=np.uint8)
        h = C.c_void_p()
        flags = (capi.W_PLANES if planes else 0) | (capi.W_PAIR if pair else 0)
        check(lib().elb_weight_create(device, ggml_type, rows, n, data.ctypes.data_as(C.c_void_p), data.nbytes, flags,
                                      C.byref(h)))
        self._h, self.type, self.device = h, ggml_type, device
        self.rows, self.n = lib().elb_weight_rows(h), lib().elb_weight_cols(h)

    @property
    def device_bytes(self):
        return lib().elb_weight_device_bytes(self._h)

    def get_rows(self, row0: int, count: int = 1) -> np.ndarray:
        out = np.empty((count, self.n), dtype=np.float32)
        check(lib().elb_get_rows(self._h, row0, count, capi.fptr(out)))
        return out

    def matvec(self, x: np.ndarray, nl: int = 4) -> np.ndarray:
        x = np.ascontiguousarray(x, dtype=np.float32)
        if x.size != self.n:
            raise ValueError("matvec: x has the wrong length")
        y = np.empty(self.rows, dtype=np.float32)
        check(lib().elb_matvec(self._h, capi.fptr(x), capi.fptr(y), nl))
        return y

    def matmul(self, x: np.ndarray, nl: int = 4) -> np.ndarray:
        x = np.ascontiguousarray(x, dtype=np.float32)
        b = x.shape[0]
        y = np.empty((b, self.rows), dtype=np.float32)
        check(lib().elb_matmul(self._h, capi.fptr(x), b, capi.fptr(y), nl))
        return y

    def limb_sums(self, x: np.ndarray, nl: int = 4):
        x = np.ascontiguousarray(x, dtype=np.float32)
        sub = 16 if self.type == synth.Q6_K else 32
        blk = 32 if self.type == synth.Q8_0 else 256
        P = np.empty((self.rows, self.n // sub, nl), dtype=np.int32)
        I = np.empty((self.rows, self.n // blk, nl), dtype=np.int32)
        J = np.empty_like(I)
        ip = lambda a: a.ctypes.data_as(C.POINTER(C.c_int32))
        check(lib().elb_limb_sums(self._h, capi.fptr(x), nl, ip(P), ip(I), ip(J)))
        return P, I, J

    def matmul_acc(self, x: np.ndarray, nl: int = 4) -> np.ndarray:
        """The int32 accumulator columns of the tensor-core limb GEMM, A[b][n/256][nl + 1][rows] (elb_matmul_acc)."""
        x = np.ascontiguousarray(x, dtype=np.float32)
        b = x.shape[0]
        A = np.empty((b, self.n // 256, nl + 1, self.rows), dtype=np.int32)
        check(lib().elb_matmul_acc(self._h, capi.fptr(x), b, nl, A.ctypes.data_as(C.POINTER(C.c_int32))))
        return A

    def close(self):
        if getattr(self, '_h', None):
            lib().elb_weight_destroy(self._h)
            self._h = None

    def __del__(self):
        self.close()


def matvec(w: Weight, x: np.ndarray, nl: int = 4) -> np.ndarray:
    """el::matvec (src/ops.h:23)"""
    return w.matvec(x, nl)


def get_row(w: Weight, row: int) -> np.ndarray:
    """el::get_row (src/ops.h:20)"""
    return w.get_rows(row, 1)[0]


def rmsnorm(x: np.ndarray, w: np.ndarray, eps: float) -> np.ndarray:
    """el::rmsnorm (src/ops.h:26) over the last axis"""
    x = np.ascontiguousarray(x, dtype=np.float32)
    w = np.ascontiguousarray(w, dtype=np.float32)
    n = x.shape[-1]
    out = np.empty_like(x)
    check(lib().elb_rmsnorm(capi.fptr(out), capi.fptr(x), capi.fptr(w), n, eps, x.size // n))
    return out


def split_limbs(x: np.ndarray, nl: int, device: int = 0):
    """k_split8 of the reference: returns (limbs[nl][b][n] int8, inv_scale[b])"""
    x = np.ascontiguousarray(np.atleast_2d(x), dtype=np.float32)
    b, n = x.shape
    limbs = np.empty((nl, b, n), dtype=np.int8)
    inv = np.empty(b, dtype=np.float32)
    check(lib().elb_split_limbs(device, capi.fptr(x), b, n, nl, limbs.ctypes.data_as(C.POINTER(C.c_int8)), capi.fptr(inv)))
    return limbs, inv


# ---- the paged cache, rotary positions and beam selection (device pointers, stream-ordered: see include/elb.h)

def _ptr(x):
    """Device address of x: a whole number, a DeviceBuffer, anything with data_ptr() (a torch tensor, say) or None. Arrays and tensors in
    pageable host memory are refused: a kernel that read there would fault."""
    if x is None or type(x) is int:
        return x
    try:  # (a decoding step makes a few of these calls per layer: every microsecond of them counts)
        p = x.data_ptr()
    except AttributeError:
        return x.ptr if isinstance(x, DeviceBuffer) else operator.index(x)
    if not getattr(x, "is_cuda", True) and not x.is_pinned():
        raise ValueError("a tensor in host memory was given where device memory is needed")
    return p


ROPE_HALF, ROPE_INTERLEAVED = 0, 1
ROPE_PLAIN, ROPE_LINEAR, ROPE_YARN, ROPE_BANDS = range(4)
KV_F16, KV_PAIR = 1, 2


def rope_config(head_dim: int = 128, dim: int | None = None, layout: int = ROPE_HALF, base: float = 1e6, scaling: int = ROPE_PLAIN,
                factor: float = 1.0, orig_ctx: float = 0.0, beta_fast: float = 32.0, beta_slow: float = 1.0, attn_factor: float = 0.0,
                low_freq: float = 1.0, high_freq: float = 4.0) -> capi.RopeConfig:
    return capi.RopeConfig(head_dim, head_dim if dim is None else dim, layout, scaling, base, factor, orig_ctx, beta_fast, beta_slow, attn_factor,
                           low_freq, high_freq)


def rope_frequencies(cfg: capi.RopeConfig):
    """(f_i, m) of a configuration (elb_rope_frequencies); host arithmetic."""
    f, m = np.empty(max(cfg.dim // 2, 1), np.float64), C.c_double()
    check(lib().elb_rope_frequencies(C.byref(cfg), f.ctypes.data_as(C.POINTER(C.c_double)), C.byref(m)))
    return f, m.value


class Rope:
    """Rotary positions (elb_rope): see rope_config for the arguments."""

    def __init__(self, head_dim: int = 128, device: int = 0, **config):
        self.config = rope_config(head_dim, **config)
        self.head_dim, h = head_dim, C.c_void_p()
        check(lib().elb_rope_create(device, C.byref(self.config), C.byref(h)))
        self._h, self._destroy, self._apply = h, lib().elb_rope_destroy, lib().elb_rope_dev

    def apply(self, x, pos, y, n: int, heads: int, ldx: int | None = None, ldy: int | None = None, norm=None, eps: float = 0.0, stream: int = 0):
        """y[n][heads] = x rotated at the positions pos[n] (elb_rope_dev); strides in floats, default the row's width."""
        w = heads * self.head_dim
        rc = self._apply(self._h, _ptr(x), w if ldx is None else ldx, _ptr(y), w if ldy is None else ldy, n, heads, _ptr(pos), _ptr(norm), eps, stream)
        if rc:
            check(rc)

    def close(self):
        if getattr(self, "_h", None):
            self._destroy(self._h)
            self._h = None

    def __del__(self):
        self.close()


class KvBatch:
    """New tokens of several sequences (elb_kv_batch): device arrays q_start[n_seq + 1], length[n_seq], table[n_seq][table_ld]."""

    def __init__(self, n_seq: int, n_tok: int, max_q: int, max_len: int, q_start, length, table, table_ld: int):
        self._keep = (q_start, length, table)
        self.n_seq, self.n_tok = n_seq, n_tok
        self._s = capi.KvBatchStruct(n_seq, n_tok, max_q, max_len, _ptr(q_start), _ptr(length), _ptr(table), table_ld)
        self._as_parameter_ = C.byref(self._s)


class KvCache:
    """A paged cache of keys and values (elb_kv). mem: device memory for the pool (kept alive here), or None."""

    def __init__(self, n_layer: int, n_head_kv: int, page: int, n_pages: int, type: int = KV_F16, mem=None, head_dim: int = 128, device: int = 0):
        h = C.c_void_p()
        self._mem, self.head_dim, self.n_head_kv = mem, head_dim, n_head_kv
        check(lib().elb_kv_create(device, n_layer, n_head_kv, head_dim, page, n_pages, type, _ptr(mem), C.byref(h)))
        self._h, self._destroy = h, lib().elb_kv_destroy
        self._append, self._attention = lib().elb_kv_append_dev, lib().elb_kv_attention_dev

    @staticmethod
    def bytes(n_layer: int, n_head_kv: int, page: int, n_pages: int, type: int = KV_F16, head_dim: int = 128) -> int:
        return lib().elb_kv_bytes(n_layer, n_head_kv, head_dim, page, n_pages, type)

    @property
    def memory(self) -> int:
        """Device address of the pool."""
        return lib().elb_kv_memory(self._h)

    def append(self, layer: int, batch: KvBatch, k, v, ldk: int, ldv: int, rope: Rope | None = None, k_norm=None, eps: float = 0.0, q=None,
               ldq: int = 0, n_head: int = 0, q_norm=None, q_out=None, ldqo: int = 0, stream: int = 0):
        """Keys and values of the batch's rows into their pages, its queries rotated into q_out (elb_kv_append_dev)."""
        rc = self._append(self._h, layer, batch._as_parameter_, rope._h if rope else None, _ptr(k), ldk, _ptr(v), ldv, _ptr(k_norm), eps, _ptr(q), ldq,
                          n_head, _ptr(q_norm), _ptr(q_out), ldqo, stream)
        if rc:
            check(rc)

    def attention_work(self, batch: KvBatch, n_head: int) -> int:
        """Bytes of working memory that attention() needs for a batch."""
        return lib().elb_kv_attention_work(self._h, batch._as_parameter_, n_head)

    def attention(self, layer: int, batch: KvBatch, q, out, n_head: int, scale: float, work, work_bytes: int, ldq: int | None = None,
                  ldo: int | None = None, stream: int = 0):
        """Attention of the batch's rows over their sequences' pages (elb_kv_attention_dev)."""
        w = n_head * self.head_dim
        rc = self._attention(self._h, layer, batch._as_parameter_, _ptr(q), w if ldq is None else ldq, n_head, scale, _ptr(out), w if ldo is None else ldo,
                             _ptr(work), work_bytes, stream)
        if rc:
            check(rc)

    def reorder(self, n: int, parent, length, table, table_ld: int, spare, length_out, table_out, taken, stream: int = 0):
        """Row r goes on from row parent[r]: tables and lengths, last pages copied where they are shared (elb_kv_reorder_dev)."""
        check(lib().elb_kv_reorder_dev(self._h, n, _ptr(parent), _ptr(length), _ptr(table), table_ld, _ptr(spare), _ptr(length_out), _ptr(table_out),
                                       _ptr(taken), stream))

    def close(self):
        if getattr(self, "_h", None):
            self._destroy(self._h)
            self._h = self._mem = None

    def __del__(self):
        self.close()


def beam_select_work(n_vocab: int, n_group: int, beams: int, k: int) -> int:
    return lib().elb_beam_select_work(n_vocab, n_group, beams, k)


def beam_select(logits, n_vocab: int, n_group: int, beams: int, scores, k: int, parent, token, score, work, work_bytes: int, ld: int | None = None,
                allowed=None, allowed_ld: int = 0, device: int = 0, stream: int = 0):
    """The k best continuations of every group of beams (elb_beam_select_dev): parent[n_group][k], token, score (double)."""
    rc = lib().elb_beam_select_dev(device, _ptr(logits), n_vocab if ld is None else ld, n_vocab, n_group, beams, _ptr(scores), _ptr(allowed),
                                   allowed_ld, k, _ptr(parent), _ptr(token), _ptr(score), _ptr(work), work_bytes, stream)
    if rc:
        check(rc)


def spec_config(spec: "synth.Spec", max_batch: int = 0, n_seq: int = 0) -> Config:
    return Config(spec.n_layer, spec.n_embd, spec.n_ff, spec.n_head, spec.n_head_kv, spec.head_dim, spec.n_vocab,
                  spec.head_dim, spec.rope_base, spec.eps, max_batch, n_seq)


def tp_unique_id() -> bytes:
    """128-byte NCCL id for Backend(tp=...): make it on one rank, hand it to the others."""
    buf = C.create_string_buffer(128)
    check(lib().elb_tp_unique_id(buf))
    return buf.raw


def tp_dims(spec: "synth.Spec", rank: int, size: int) -> dict:
    """This rank's share of the model: heads, FFN range [f0, f1), vocabulary rows [v0, v1). Host arithmetic only."""
    cfg = spec_config(spec)
    h, hkv = C.c_int(), C.c_int()
    f0, f1, v0, v1 = C.c_int64(), C.c_int64(), C.c_int64(), C.c_int64()
    check(lib().elb_tp_dims(C.byref(cfg), rank, size, C.byref(h), C.byref(hkv), C.byref(f0), C.byref(f1), C.byref(v0),
                            C.byref(v1)))
    return {"n_head": h.value, "n_head_kv": hkv.value, "f0": f0.value, "f1": f1.value, "v0": v0.value, "v1": v1.value}


def tp_shard(spec: "synth.Spec", rank: int, size: int, role: str, t: int, rows: int, n: int, data: np.ndarray):
    """Rank `rank`'s cut of one tensor of the whole model: (rows, n, bytes). Host arithmetic only."""
    cfg = spec_config(spec)
    data = np.ascontiguousarray(data, dtype=np.uint8).reshape(-1)
    orows, on, nb = C.c_int64(), C.c_int64(), C.c_size_t()
    rid = synth.ROLE_ID[role]
    check(lib().elb_tp_shard_shape(C.byref(cfg), rank, size, rid, t, rows, n, C.byref(orows), C.byref(on), C.byref(nb)))
    out = np.empty(nb.value, dtype=np.uint8)
    check(lib().elb_tp_shard_copy(C.byref(cfg), rank, size, rid, t, rows, n, data.ctypes.data_as(C.c_void_p), data.nbytes,
                                  out.ctypes.data_as(C.c_void_p), out.nbytes))
    return orows.value, on.value, out


class Backend:
    """el::Backend (src/model.h:42-51) on the CUDA library: cfg(), n_ctx(), name(), eval(tokens, pos0) -> logits."""

    def __init__(self, spec: "synth.Spec", tensors, n_ctx: int, device: int = 0, max_batch: int = 0, tp=None,
                 n_seq: int = 0, pages=None):
        """tp = (rank, size, id) makes this process rank `rank` of a tensor-parallel group of `size` GPUs; `id` is the
        128-byte value of tp_unique_id() made on one rank and given to all. `tensors` are the whole model's on every
        rank; eval must then be called by all ranks with the same arguments. pages = (page, n_pages, type): a paged cache
        shared by all sequences (elb_model_set_pages)."""
        self.spec = spec
        self._cfg = spec_config(spec, max_batch, n_seq)
        self._n_ctx = n_ctx
        h = C.c_void_p()
        if tp is None or tp[1] == 1:
            check(lib().elb_model_create(C.byref(self._cfg), n_ctx, device, C.byref(h)))
        else:
            rank, size, ident = tp
            buf = C.create_string_buffer(bytes(ident), 128)
            check(lib().elb_model_create_tp(C.byref(self._cfg), n_ctx, device, rank, size, buf, C.byref(h)))
        self._h = h
        try:
            if pages is not None:
                check(lib().elb_model_set_pages(h, *pages))
            keep = []
            for role, layer, t, rows, n, data in tensors:
                data = np.ascontiguousarray(data, dtype=np.uint8)
                keep.append(data)  # bytes must stay valid until finalize
                check(lib().elb_model_set_tensor(h, synth.ROLE_ID[role], max(layer, 0), t, rows, n,
                                                 data.ctypes.data_as(C.c_void_p), data.nbytes))
            check(lib().elb_model_finalize(h))
        except Exception:
            self.close()
            raise
        self._logits_host = None

    @classmethod
    def from_gguf(cls, path: str, n_ctx: int, device: int = 0, max_batch: int = 0, n_seq: int = 0, tp=None):
        """The model of a GGUF file, read and uploaded by the library itself (elb_model_load_gguf); tp = (rank, size,
        id) makes this process one rank of a tensor-parallel group that loads the same file (elb_model_load_gguf_tp)."""
        h = C.c_void_p()
        if tp is None:
            check(lib().elb_model_load_gguf(os.fsencode(path), n_ctx, device, max_batch, n_seq, C.byref(h)))
        else:
            rank, size, ident = tp
            buf = C.create_string_buffer(bytes(ident), 128)
            check(lib().elb_model_load_gguf_tp(os.fsencode(path), n_ctx, device, max_batch, n_seq, rank, size, buf, C.byref(h)))
        self = cls.__new__(cls)
        self._h, self._n_ctx, self._logits_host = h, n_ctx, None
        self._cfg = Config()
        check(lib().elb_model_config(h, C.byref(self._cfg)))
        c = self._cfg
        self.spec = synth.Spec(name=os.path.basename(path), n_layer=c.n_layer, n_embd=c.n_embd, n_ff=c.n_ff, n_head=c.n_head,
                               n_head_kv=c.n_head_kv, n_vocab=c.n_vocab, layout="gguf", head_dim=c.head_dim,
                               rope_base=c.rope_base, eps=c.eps)
        return self

    def cfg(self):
        return self._cfg

    def n_ctx(self):
        return self._n_ctx

    def name(self):
        return "cuda-b200"

    def eval(self, tokens, pos0: int, want_logits: bool = True, out: np.ndarray | None = None):
        tokens = np.ascontiguousarray(tokens, dtype=np.int32)
        logits = None
        if want_logits:
            logits = out if out is not None else np.empty(self.spec.n_vocab, dtype=np.float32)
        check(lib().elb_model_eval(self._h, tokens.ctypes.data_as(C.POINTER(C.c_int32)), tokens.size, pos0,
                                   logits.ctypes.data_as(C.c_void_p) if want_logits else None))
        return logits

    def eval_top(self, tokens, pos0: int, k: int = 1, allowed=None):
        """eval with the logits reduced on the device: (ids[k], logits[k], log-sum-exp) of the last token, ids ordered by
        (logit descending, id ascending); logprob of ids[i] = logits[i] - lse. allowed: boolean mask over the vocabulary
        (constrained decoding): only allowed tokens are picked, the log-sum-exp still covers all."""
        tokens = np.ascontiguousarray(tokens, dtype=np.int32)
        ids, vals, lse = np.empty(k, np.int32), np.empty(k, np.float32), C.c_double()
        i32 = C.POINTER(C.c_int32)
        if allowed is None:
            check(lib().elb_model_eval_top(self._h, tokens.ctypes.data_as(i32), tokens.size, pos0, k, ids.ctypes.data_as(i32),
                                           capi.fptr(vals), C.byref(lse)))
        else:
            bits = np.packbits(np.asarray(allowed, dtype=bool), bitorder="little")
            words = np.zeros((self.spec.n_vocab + 31) // 32 * 4, np.uint8)
            words[:bits.size] = bits
            check(lib().elb_model_eval_top_masked(self._h, tokens.ctypes.data_as(i32), tokens.size, pos0, k,
                                                  words.ctypes.data_as(C.c_void_p), ids.ctypes.data_as(i32), capi.fptr(vals),
                                                  C.byref(lse)))
        return ids, vals, lse.value

    def eval_batch(self, tokens, seq, pos, want=None, want_logits: bool = True):
        """Rows of several sequences in one pass: row i is tokens[i] at position pos[i] of sequence seq[i] (n_seq given at
        construction). Returns one row of logits per wanted row (want: boolean mask, default all rows), or None."""
        tokens = np.ascontiguousarray(tokens, dtype=np.int32)
        seq = np.ascontiguousarray(seq, dtype=np.int32)
        pos = np.ascontiguousarray(pos, dtype=np.int32)
        n = tokens.size
        w = None if want is None else np.ascontiguousarray(want, dtype=np.uint8)
        n_out = n if w is None else int(np.count_nonzero(w))
        out = np.empty((n_out, self.spec.n_vocab), dtype=np.float32) if want_logits else None
        i32 = C.POINTER(C.c_int32)
        check(lib().elb_model_eval_batch(self._h, n, tokens.ctypes.data_as(i32), seq.ctypes.data_as(i32), pos.ctypes.data_as(i32),
                                         w.ctypes.data_as(C.c_void_p) if w is not None else None,
                                         out.ctypes.data_as(C.c_void_p) if want_logits else None))
        return out

    def eval_batch_top(self, tokens, seq, pos, k: int = 1, want=None):
        """eval_batch with every wanted row reduced on the device: (ids[R][k], logits[R][k], lse[R])."""
        tokens = np.ascontiguousarray(tokens, dtype=np.int32)
        seq = np.ascontiguousarray(seq, dtype=np.int32)
        pos = np.ascontiguousarray(pos, dtype=np.int32)
        n = tokens.size
        w = None if want is None else np.ascontiguousarray(want, dtype=np.uint8)
        R = n if w is None else int(np.count_nonzero(w))
        ids, vals, lse = np.empty((R, k), np.int32), np.empty((R, k), np.float32), np.empty(R, np.float64)
        i32 = C.POINTER(C.c_int32)
        check(lib().elb_model_eval_batch_top(self._h, n, tokens.ctypes.data_as(i32), seq.ctypes.data_as(i32), pos.ctypes.data_as(i32),
                                             w.ctypes.data_as(C.c_void_p) if w is not None else None, k, ids.ctypes.data_as(i32),
                                             capi.fptr(vals), lse.ctypes.data_as(C.POINTER(C.c_double))))
        return ids, vals, lse

    def eval_batch_beam(self, tokens, seq, pos, scores, beams: int, k: int, want=None):
        """eval_batch with beam search's selection on the device: the wanted rows are groups of `beams` rows with scores[R] so far;
        returns (parent[G][k], token[G][k], score[G][k]), parents counted over the wanted rows (elb_model_eval_batch_beam)."""
        tokens = np.ascontiguousarray(tokens, dtype=np.int32)
        seq = np.ascontiguousarray(seq, dtype=np.int32)
        pos = np.ascontiguousarray(pos, dtype=np.int32)
        scores = np.ascontiguousarray(scores, dtype=np.float64)
        w = None if want is None else np.ascontiguousarray(want, dtype=np.uint8)
        R = tokens.size if w is None else int(np.count_nonzero(w))
        if scores.size != R or beams < 1 or R % beams:
            raise ValueError("eval_batch_beam: one score per wanted row, and whole groups of beams")
        G, i32, f64 = R // beams, C.POINTER(C.c_int32), C.POINTER(C.c_double)
        parent, token, score = np.empty((G, max(k, 0)), np.int32), np.empty((G, max(k, 0)), np.int32), np.empty((G, max(k, 0)), np.float64)
        check(lib().elb_model_eval_batch_beam(self._h, tokens.size, tokens.ctypes.data_as(i32), seq.ctypes.data_as(i32), pos.ctypes.data_as(i32),
                                              w.ctypes.data_as(C.c_void_p) if w is not None else None, G, beams, scores.ctypes.data_as(f64), k,
                                              parent.ctypes.data_as(i32), token.ctypes.data_as(i32), score.ctypes.data_as(f64)))
        return parent, token, score

    def reorder(self, seq, parent):
        """Sequence seq[i] goes on from the state of parent[i], all at once (elb_model_reorder; paged models)."""
        seq, parent = np.ascontiguousarray(seq, dtype=np.int32), np.ascontiguousarray(parent, dtype=np.int32)
        if seq.size != parent.size:
            raise ValueError("reorder: one parent per sequence")
        i32 = C.POINTER(C.c_int32)
        check(lib().elb_model_reorder(self._h, seq.size, seq.ctypes.data_as(i32), parent.ctypes.data_as(i32)))

    def drop(self, seq: int):
        """Gives a sequence's pages back (elb_model_drop; paged models)."""
        check(lib().elb_model_drop(self._h, seq))

    def free_pages(self) -> int:
        n = C.c_int32()
        check(lib().elb_model_free_pages(self._h, C.byref(n)))
        return n.value

    def eval_steps(self, tokens, pos0: int) -> float:
        """Single-token steps back to back, logits left on the device; returns the device time in ms."""
        tokens = np.ascontiguousarray(tokens, dtype=np.int32)
        ms = C.c_float()
        check(lib().elb_model_eval_steps(self._h, tokens.ctypes.data_as(C.POINTER(C.c_int32)), tokens.size, pos0,
                                         C.byref(ms)))
        return ms.value

    def last_eval_stats(self):
        ms, n = C.c_float(), C.c_int64()
        check(lib().elb_model_last_eval_stats(self._h, C.byref(ms), C.byref(n)))
        return ms.value, n.value

    def hidden(self):
        out = np.empty(self.spec.n_embd, dtype=np.float32)
        check(lib().elb_model_hidden(self._h, capi.fptr(out)))
        return out

    @property
    def weight_bytes(self):
        return lib().elb_model_weight_bytes(self._h)

    @property
    def kv_bytes_per_token(self):
        return lib().elb_model_kv_bytes_per_token(self._h)

    def close(self):
        if getattr(self, "_h", None):
            lib().elb_model_destroy(self._h)
            self._h = None

    def __del__(self):
        self.close()
