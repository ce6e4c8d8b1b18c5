"""Single operators of the C ABI (``neko_op_*``) on torch CUDA tensors. torch is only the device allocator and
stream here; the arithmetic is the library's."""
import ctypes as C
import struct

from . import NekoError, check, lib


def _ptr(t):
    if t is None:
        return None
    if not t.is_cuda or not t.is_contiguous():
        raise NekoError("ops take contiguous CUDA tensors")
    return C.c_void_p(t.data_ptr())


def _stream():
    import torch
    return C.c_void_p(torch.cuda.current_stream().cuda_stream)


def row_bytes(fmt, cols):
    """quantRowBytes (quant.cpp:199-208)."""
    return int(lib().neko_row_bytes(fmt, cols))


def quantize(fmt, w, transpose_f16=False):
    """quantizeMatrix (quant.cpp:255-279) on the GPU. w: [rows][cols] float32 CUDA tensor (or [cols][rows] with
    transpose_f16, the Conv1D layout). Returns [rows][row_bytes] uint8."""
    import torch
    if transpose_f16:
        cols, rows = w.shape
    else:
        rows, cols = w.shape
    out = torch.zeros((rows, row_bytes(fmt, cols)), dtype=torch.uint8, device=w.device)
    ld = w.shape[1]
    check(lib().neko_op_quantize(fmt, _ptr(w), rows, cols, ld, 1 if transpose_f16 else 0, _ptr(out), _stream()),
          "quantize")
    return out


def dequantize(fmt, q, cols):
    """QMatrix::dequantizeRow for every row (quant.cpp:230-253)."""
    import torch
    out = torch.empty((q.shape[0], cols), dtype=torch.float32, device=q.device)
    check(lib().neko_op_dequantize(fmt, _ptr(q), q.shape[0], cols, _ptr(out), _stream()), "dequantize")
    return out


def matmul(fmt, x, q, K, bias=None, y=None, y_stride=None, n_off=0, flags=0):
    """cpu::matmul semantics (cpu_ops.h:17-23): y[t][n_off + n] (+)= act(x[t] . W[n] + bias[n])."""
    import torch
    T = x.numel() // K
    rows = q.shape[0]
    y_stride = rows if y_stride is None else y_stride
    if y is None:
        y = torch.zeros((T, y_stride), dtype=torch.float32, device=x.device)
    if bias is not None:
        flags |= 4
    check(lib().neko_op_matmul(fmt, _ptr(x), T, K, _ptr(q), rows, _ptr(bias), _ptr(y), y_stride, n_off, flags,
                               _stream()), "matmul")
    return y


def matmul_fused(fmt, x, q, K, rows, norm=0, gamma=None, beta=None, eps=1e-6, swiglu=False, bias=None, y=None,
                 y_stride=None, n_off=0, flags=0):
    """Norm prologue (0 none, 1 RMSNorm, 2 LayerNorm) + matmul, or the SwiGLU pair (q holds 2 * rows rows)."""
    import torch
    T = x.numel() // K
    y_stride = rows if y_stride is None else y_stride
    if y is None:
        y = torch.zeros((T, y_stride), dtype=torch.float32, device=x.device)
    if bias is not None:
        flags |= 4
    check(lib().neko_op_matmul_fused(fmt, _ptr(x), T, K, _ptr(q), rows, norm, _ptr(gamma), _ptr(beta), eps,
                                     1 if swiglu else 0, _ptr(bias), _ptr(y), y_stride, n_off, flags, _stream()),
          "matmul_fused")
    return y


def norm(x, gamma, beta=None, eps=1e-6):
    """cpu::rmsNorm (beta None) / cpu::layerNorm over the last dimension."""
    import torch
    C_ = x.shape[-1]
    y = torch.empty_like(x)
    check(lib().neko_op_norm(_ptr(x), _ptr(y), _ptr(gamma), _ptr(beta), x.numel() // C_, C_, eps, _stream()), "norm")
    return y


def softmax(x):
    import torch
    C_ = x.shape[-1]
    y = torch.empty_like(x)
    check(lib().neko_op_softmax(_ptr(x), _ptr(y), x.numel() // C_, C_, _stream()), "softmax")
    return y


def argmax(x):
    import torch
    C_ = x.shape[-1]
    out = torch.empty(x.numel() // C_, dtype=torch.int32, device=x.device)
    check(lib().neko_op_argmax(_ptr(x), x.numel() // C_, C_, _ptr(out), _stream()), "argmax")
    return out


def sample(logits, u, temperature=0.8, top_k=40, top_p=0.95, repeat_penalty=1.1, repeat_last_n=64, history=None,
           hist_len=None):
    """Sampler::sample per row of logits [rows][V] (modified in place by the repetition penalty) with the uniform
    draws u [rows] (float64); history [rows][S] int32 with hist_len [rows] valid tokens. Returns int32 [rows]."""
    import torch
    from . import Sampling
    rows, V = logits.shape
    out = torch.empty(rows, dtype=torch.int32, device=logits.device)
    sp = Sampling(temperature, top_k, top_p, repeat_penalty, repeat_last_n)
    check(lib().neko_op_sample(_ptr(logits), rows, V, _ptr(history) if history is not None else None,
                               _ptr(hist_len) if hist_len is not None else None,
                               history.shape[1] if history is not None else 0,
                               _ptr(u) if u is not None else None, C.byref(sp), _ptr(out), _stream()), "sample")
    return out


def fp8_block_dequant(codes, scales):
    """An FP8 (E4M3) checkpoint weight as f32 (TensorStore::toF32, tensor_store.cpp:543-571, 578-590): codes
    uint8 [rows][cols], scales float32 [sR][sC] (the "_scale_inv" / "_scale" tensor; 1 x 1 per tensor), both CUDA
    tensors. Returns float32 [rows][cols]."""
    import torch
    rows, cols = codes.shape
    s2 = scales.reshape(scales.shape[0] if scales.dim() else 1, -1)
    out = torch.empty((rows, cols), dtype=torch.float32, device=codes.device)
    check(lib().neko_op_fp8_block_dequant(_ptr(codes), rows, cols, _ptr(scales), s2.shape[0], s2.shape[1], _ptr(out),
                                          _stream()), "fp8_block_dequant")
    return out


def attention(q, q_stride, k_cache, v_cache, T, n_head, n_kv, hd, pos0):
    """cpu::attention (cpu_ops.cpp:544-575) over engine-layout caches [ctx][n_kv * hd] (int16/uint16 f16 bits)."""
    import torch
    out = torch.empty((T, n_head * hd), dtype=torch.float32, device=q.device)
    check(lib().neko_op_attention(_ptr(q), q_stride, _ptr(k_cache), _ptr(v_cache), _ptr(out), T, n_head, n_kv, hd,
                                  pos0, _stream()), "attention")
    return out


# ------------------------------------------------------------------ paged key/value cache
# neko_paged_cache, neko_paged_append_args and neko_paged_attention_args (include/neko_cuda.h)
_CACHE = "5P3q8i"
_APPEND = struct.Struct("@" + _CACHE + "4P8q5P7if")
_ATTEND = struct.Struct("@" + _CACHE + "2P4q4P5i2fi")
_TREE = struct.Struct("@2P2i")
_PLANES = struct.Struct("@3P5q8i")
_SAMPLE = struct.Struct("@8Pq4i3fi")
_types = {}


def _setup():
    """neko_type of each dtype (uint8 and float8_e4m3fn both hold E4M3 codes) and the entries, on first use."""
    import torch
    l = lib()
    _types.update({torch.float32: 0, torch.float16: 1, torch.bfloat16: 2, torch.float8_e4m3fn: 3, torch.uint8: 3,
                   "f32": torch.float32, "i32": torch.int32, "append": l.neko_op_paged_append,
                   "attend": l.neko_op_paged_attention, "i64": torch.int64, "f64": torch.float64,
                   "tree_append": l.neko_op_paged_tree_append, "tree_attend": l.neko_op_paged_tree_attention,
                   "masks": l.neko_op_tree_masks, "accept": l.neko_op_tree_accept, "compact": l.neko_op_paged_compact,
                   "copy": l.neko_op_paged_copy, "sample": l.neko_op_sample_rows, "device": torch.cuda.current_device,
                   "stream": getattr(torch._C, "_cuda_getCurrentRawStream", None) or
                   (lambda i: torch.cuda.current_stream(i).cuda_stream)})
    return _types


def _rows(t, what, dtype, shape, dev):
    """(pointer, token stride, head stride) of [tokens][heads][hd] rows."""
    if t.dtype is not dtype or t.shape != shape or t.get_device() != dev:
        raise NekoError(f"{what}: {dtype} {list(shape)} on cuda:{dev}, got {t.dtype} {list(t.shape)} on {t.device}")
    st = t.stride()
    if st[2] != 1:
        raise NekoError(f"{what}: the last dimension is contiguous")
    return t.data_ptr(), st[0], st[1]


def _vector(t, what, dtype, n, dev):
    """Pointer of n contiguous numbers, NULL for None."""
    if t is None:
        return 0
    if t.dtype is not dtype or t.numel() != n or t.get_device() != dev or not t.is_contiguous():
        raise NekoError(f"{what}: {n} contiguous {dtype} on cuda:{dev}")
    return t.data_ptr()


def _cache(k_pages, v_pages, k_scale, v_scale, table, types):
    """The fields of neko_paged_cache, then n_seq, n_kv, head dim and device index."""
    dev, sh, st, dt = k_pages.get_device(), k_pages.shape, k_pages.stride(), k_pages.dtype
    if dev < 0 or len(sh) != 4 or v_pages.shape != sh or v_pages.stride() != st or v_pages.get_device() != dev or \
            v_pages.dtype is not dt or dt not in types:
        raise NekoError("paged cache: k_pages and v_pages are alike [pages][kv heads][page][head_dim] CUDA tensors "
                        "(float16, float8_e4m3fn or uint8)")
    pages, n_kv, ps, hd = sh
    if st[3] != 1 or st[2] != hd or (st[1] != ps * hd and n_kv > 1):
        raise NekoError("paged cache: a page is contiguous")
    type_ = types[dt]
    ks = vs = sst = 0
    if type_ == 3:
        if k_scale is None or v_scale is None:
            raise NekoError("paged cache: 8-bit pages need k_scale and v_scale")
        sst = k_scale.stride()[0]
        for t in (k_scale, v_scale):
            s2 = t.stride()
            if t.shape != (pages, n_kv) or t.dtype is not types["f32"] or t.get_device() != dev or s2[0] != sst or \
                    (n_kv > 1 and s2[1] != 1):
                raise NekoError("paged cache: scales are alike [pages][kv heads] float32")
        ks, vs = k_scale.data_ptr(), v_scale.data_ptr()
    tsh, tst = table.shape, table.stride()
    if len(tsh) != 2 or table.dtype is not types["i32"] or table.get_device() != dev or (tsh[1] > 1 and tst[1] != 1):
        raise NekoError("paged cache: the table is [sequences][pages] int32")
    n_seq, width = tsh
    if types["device"]() != dev:
        raise NekoError(f"paged cache: the tensors are on cuda:{dev}, which is not the current device")
    return (k_pages.data_ptr(), v_pages.data_ptr(), ks, vs, table.data_ptr(), st[0] if pages > 1 else n_kv * ps * hd, sst,
            tst[0] if n_seq > 1 else width, type_, n_seq, width, pages, n_kv, ps, hd, 0), n_seq, n_kv, hd, dev


def rope_table(positions, rot, theta, scaling="none", factor=1.0, original=0, beta_fast=32.0, beta_slow=1.0,
               device="cuda"):
    """The (cos, sin) table [positions][rot / 2][2] of paged_append, computed in double like Qwen3Model::ropeTable
    (qwen3_model.cpp) and rounded once. Pair j turns by pos * theta^(-2j / rot). Longer contexts (factor times the
    `original` positions a model was trained on):
      "linear" positions divided by factor;
      "ntk"    theta raised to theta * factor^(rot / (rot - 2)), so the slowest pair is slowed by factor;
      "yarn"   pairs that turn more than beta_fast times over `original` positions keep their speed, those below
               beta_slow turns are slowed by factor, a linear ramp between (its ends in whole pairs, in [0, rot - 1]; the
               upper one may lie past the last pair, which then is slowed in part), and cos and sin are multiplied by
               0.1 ln(factor) + 1 (YaRN, Peng et al. 2023)."""
    import math

    import numpy as np
    import torch
    if rot <= 0 or rot % 8 or positions <= 0 or theta <= 0 or factor < 1:
        raise NekoError("rope_table: rot a positive multiple of 8, positions and theta positive, factor >= 1")
    half = rot // 2
    j = np.arange(half, dtype=np.float64)
    gain = 1.0
    if scaling == "ntk":
        theta = theta * factor ** (rot / (rot - 2))
    freq = theta ** (-j / half)
    if scaling == "linear":
        freq = freq / factor
    elif scaling == "yarn":
        if original <= 0:
            raise NekoError("rope_table: yarn needs the original context length")
        pair = lambda turns: half * math.log(original / (turns * 2 * math.pi)) / math.log(theta)  # noqa: E731
        low, high = max(math.floor(pair(beta_fast)), 0), min(math.ceil(pair(beta_slow)), rot - 1)
        slow = np.clip((j - low) / max(high - low, 1e-3), 0, 1)
        freq = freq * (1 - slow) + freq / factor * slow
        gain = 0.1 * math.log(factor) + 1.0
    elif scaling not in ("none", "ntk"):
        raise NekoError(f"rope_table: unknown scaling {scaling!r}")
    ang = np.arange(positions, dtype=np.float64)[:, None] * freq
    return torch.from_numpy(np.stack([np.cos(ang) * gain, np.sin(ang) * gain], -1).astype(np.float32)).to(device)


def paged_append(k, v, k_pages, v_pages, table, start, k_scale=None, v_scale=None, q_start=None, max_new=1, q=None,
                 cs=None, interleaved=False, q_gain=None, k_gain=None, eps=1e-6, q_out=None, depth=None):
    """neko_op_paged_append: k, v [tokens][kv heads][hd] (any token and head stride) go to the pages, after the
    per-head norm (k_gain) and the rotation by cs (rope_table) of k. Sequence s's rows are q_start[s] ..
    q_start[s + 1] - 1 (q_start None: row s) and go to positions start[s], start[s] + 1, ..; at most max_new per
    sequence. depth [tokens] (neko_op_paged_tree_append): the new tokens are nodes of a tree, turned by start[s] + depth
    instead of their places. Returns q with its norm (q_gain) and rotation applied (into q_out, which may be q; a new tensor when
    None), or None without q."""
    types = _types or _setup()
    fields, n_seq, n_kv, hd, dev = _cache(k_pages, v_pages, k_scale, v_scale, table, types)
    dt, tokens = k.dtype, k.shape[0]
    shape = (tokens, n_kv, hd)
    kp = _rows(k, "paged_append k", dt, shape, dev)
    vp = _rows(v, "paged_append v", dt, shape, dev)
    qp = op = (0, 0, 0)
    heads = 0
    if q is not None:
        heads = q.shape[1]
        shape = (tokens, heads, hd)
        qp = _rows(q, "paged_append q", dt, shape, dev)
        if q_out is None:
            q_out = q.new_empty(shape)
        op = _rows(q_out, "paged_append q_out", dt, shape, dev)
    rot = rows = csp = 0
    if cs is not None:
        rows, half, two = cs.shape
        rot = 2 * half
        if two != 2:
            raise NekoError("paged_append: cs is [positions][rot / 2][2]")
        csp = _vector(cs, "paged_append cs", types["f32"], rows * rot, dev)
    i32, f32 = types["i32"], types["f32"]
    args = _APPEND.pack(*fields, qp[0], kp[0], vp[0], op[0], *qp[1:], *kp[1:], *vp[1:], *op[1:],
                        _vector(start, "paged_append start", i32, n_seq, dev),
                        _vector(q_start, "paged_append q_start", i32, n_seq + 1, dev), csp,
                        _vector(q_gain, "paged_append q_gain", f32, hd, dev),
                        _vector(k_gain, "paged_append k_gain", f32, hd, dev),
                        types.get(dt, -1), tokens, heads, max_new, rot, rows, 1 if interleaved else 0, eps)
    if depth is None:
        rc = types["append"](args, types["stream"](dev))
    else:
        rc = types["tree_append"](args, _vector(depth, "paged_append depth", i32, tokens, dev), types["stream"](dev))
    if rc:
        check(rc, "paged_append")
    return q_out if q is not None else None


def paged_attention(q, k_pages, v_pages, table, kv_len, k_scale=None, v_scale=None, q_start=None, max_new=1,
                    scale=None, softcap=0.0, window=0, slopes=None, prefix=None, out=None):
    """neko_op_paged_attention: q [tokens][heads][hd] over the cached keys and values; kv_len [sequences] counts the
    new tokens, which are in the cache already. scale: 1 / sqrt(hd) when None; softcap, window, slopes [heads] and
    prefix [sequences] as the header defines them. Returns out (shaped and typed like q)."""
    return _attend("paged_attention", q, k_pages, v_pages, table, kv_len, k_scale, v_scale, q_start, max_new, scale, softcap,
                   window, slopes, prefix, out)


def _attend(what, q, k_pages, v_pages, table, kv_len, k_scale, v_scale, q_start, max_new, scale, softcap, window, slopes, prefix,
            out, mask=None, depth=None):
    types = _types or _setup()
    fields, n_seq, n_kv, hd, dev = _cache(k_pages, v_pages, k_scale, v_scale, table, types)
    dt, shape = q.dtype, q.shape
    if len(shape) != 3 or shape[2] != hd:
        raise NekoError(f"{what} q: [tokens][heads][head_dim] rows")
    qp = _rows(q, what + " q", dt, shape, dev)
    if out is None:
        out = q.new_empty(shape)
    op = _rows(out, what + " out", dt, shape, dev)
    i32 = types["i32"]
    args = _ATTEND.pack(*fields, qp[0], op[0], *qp[1:], *op[1:], _vector(kv_len, what + " kv_len", i32, n_seq, dev),
                        _vector(q_start, what + " q_start", i32, n_seq + 1, dev),
                        _vector(slopes, what + " slopes", types["f32"], shape[1], dev),
                        _vector(prefix, what + " prefix", i32, n_seq, dev), types.get(dt, -1), shape[0], shape[1],
                        max_new, window, hd ** -0.5 if scale is None else scale, softcap, 0)
    if mask is None:
        rc = types["attend"](args, types["stream"](dev))
    else:
        words = mask.shape[1]
        tree = _TREE.pack(_vector(mask, what + " mask", types["i64"], shape[0] * words, dev),
                          _vector(depth, what + " depth", i32, shape[0], dev), words, 0)
        rc = types["tree_attend"](args, tree, types["stream"](dev))
    if rc:
        check(rc, what)
    return out


# ------------------------------------------------------------------ drafted tokens
def paged_tree_attention(q, k_pages, v_pages, table, kv_len, mask, depth=None, k_scale=None, v_scale=None, q_start=None,
                         max_new=1, scale=None, softcap=0.0, window=0, slopes=None, out=None):
    """neko_op_paged_tree_attention: paged_attention for the nodes of trees of drafted tokens, which are in the cache already:
    each sees the keys before the tree and the nodes of its mask (int64 [tokens][words], 64 nodes a word, as tree_masks
    gives it); positions (window, slopes) go by depth [tokens]. Returns out (shaped and typed like q)."""
    if getattr(mask, "ndim", 0) != 2:
        raise NekoError("paged_tree_attention: a mask [tokens][words]")
    return _attend("paged_tree_attention", q, k_pages, v_pages, table, kv_len, k_scale, v_scale, q_start, max_new, scale, softcap,
                   window, slopes, None, out, mask, depth)


def _on_device(t, what, types):
    dev = t.get_device()
    if dev < 0 or types["device"]() != dev:
        raise NekoError(f"{what}: CUDA tensors on the current device")
    return dev


def tree_masks(parent, q_start, max_new):
    """neko_op_tree_masks: parent int32 [tokens] (each node's parent, counted from its sequence's first node; no earlier node: a
    root), sequence s's nodes at q_start[s] .. q_start[s + 1] - 1, at most max_new. Returns mask int64
    [tokens][ceil(max_new / 64)] (bit j: node j is the node itself or an ancestor) and depth int32 [tokens]. Rows of no
    sequence are zeros."""
    types = _types or _setup()
    dev, tokens, i32 = _on_device(parent, "tree_masks", types), parent.numel(), types["i32"]
    n_seq, words = q_start.numel() - 1, max((max_new + 63) // 64, 1)
    mask, depth = parent.new_empty((tokens, words), dtype=types["i64"]), parent.new_empty(tokens)
    rc = types["masks"](_vector(parent, "tree_masks parent", i32, tokens, dev), _vector(q_start, "tree_masks q_start", i32, n_seq + 1, dev),
                        n_seq, tokens, max_new, mask.data_ptr(), words, depth.data_ptr(), types["stream"](dev))
    if rc:
        check(rc, "tree_masks")
    return (mask, depth) if n_seq and max_new else (mask.zero_(), depth.zero_())


def tree_accept(chosen, draft, parent, q_start, max_new):
    """neko_op_tree_accept: walks each sequence's tree (parent, q_start, max_new as in tree_masks) from its node 0 to the lowest
    child whose draft is the token chosen at the node, and so on; chosen, draft int32 [tokens]. Returns path int32
    [sequences][max_new] (the nodes, then zeros), count int32 [sequences] and token int32 [sequences], the one chosen at the
    last of them (a sequence without nodes: 0 and -1)."""
    types = _types or _setup()
    dev, tokens, i32 = _on_device(parent, "tree_accept", types), parent.numel(), types["i32"]
    n_seq = q_start.numel() - 1
    if n_seq < 0 or max_new < 0:
        raise NekoError("tree_accept: q_start [sequences + 1], max_new of zero or more")
    path, count, token = parent.new_empty((n_seq, max_new)), parent.new_empty(n_seq), parent.new_empty(n_seq)
    rc = types["accept"](_vector(chosen, "tree_accept chosen", i32, tokens, dev), _vector(draft, "tree_accept draft", i32, tokens, dev),
                         _vector(parent, "tree_accept parent", i32, tokens, dev), _vector(q_start, "tree_accept q_start", i32, n_seq + 1, dev),
                         n_seq, tokens, max_new, path.data_ptr(), count.data_ptr(), token.data_ptr(), types["stream"](dev))
    if rc:
        check(rc, "tree_accept")
    return path, count, token


def _planes(pool, scale, table, what, types):
    """The fields of neko_paged_planes and the device index; pool [..][pages][kv heads][page][hd], any uniform planes."""
    dev, sh, st = _on_device(pool, what, types), pool.shape, pool.stride()
    type_ = types.get(pool.dtype, -1)
    if len(sh) < 4:
        raise NekoError(f"{what}: the pool is [planes ..][pages][kv heads][page][head_dim]")
    pages, n_kv, ps, hd = sh[-4:]
    if st[-1] != 1 or st[-2] != hd or (st[-3] != ps * hd and n_kv > 1):
        raise NekoError(f"{what}: a page is contiguous")

    def uniform(shape, stride, name):
        """Planes and their stride, leading dimensions taken together."""
        n, step = 1, 0
        for s, d in zip(reversed(shape), reversed(stride)):
            if s == 1:
                continue
            if n > 1 and d != n * step:
                raise NekoError(f"{what}: the {name}'s planes are not a constant step apart")
            if n == 1:
                step = d
            n *= s
        return n, step

    planes, step = uniform(sh[:-4], st[:-4], "pool")
    sp = plane = page = 0
    if type_ == 3:
        if scale is None or scale.dtype is not types["f32"] or scale.get_device() != dev or scale.shape != sh[:-2] or \
                (n_kv > 1 and scale.stride(-1) != 1):
            raise NekoError(f"{what}: 8-bit pages need scales float32 [planes ..][pages][kv heads]")
        plane, page = uniform(sh[:-4], scale.stride()[:-2], "scales")[1], scale.stride(-2) if pages > 1 else n_kv
        sp = scale.data_ptr()
    n_seq = width = tp = ts = 0
    if table is not None:
        tsh, tst = table.shape, table.stride()
        if len(tsh) != 2 or table.dtype is not types["i32"] or table.get_device() != dev or (tsh[1] > 1 and tst[1] != 1):
            raise NekoError(f"{what}: the table is [sequences][pages] int32")
        (n_seq, width), tp = tsh, table.data_ptr()
        ts = tst[0] if n_seq > 1 else width
    return _PLANES.pack(pool.data_ptr(), sp, tp, step, st[-4] if pages > 1 else n_kv * ps * hd, plane, page, ts, type_, planes,
                        n_seq, width, pages, n_kv, ps, hd), n_seq, dev


def paged_compact(pool, table, start, path, count, scale=None):
    """neko_op_paged_compact: in every plane of pool [planes ..][pages][kv heads][page][hd] (scale [planes ..][pages][kv heads] with
    8-bit pages), token start[s] + path[s][k] becomes token start[s] + k, k < count[s]: what tree_accept leaves of a tree. Paths
    [sequences][width] int32 ascend."""
    types = _types or _setup()
    args, n_seq, dev = _planes(pool, scale, table, "paged_compact", types)
    i32 = types["i32"]
    if path.dtype is not i32 or path.dim() != 2 or path.shape[0] != n_seq or path.get_device() != dev or \
            (path.shape[1] > 1 and path.stride(1) != 1):
        raise NekoError("paged_compact path: int32 [sequences][width]")
    width = path.shape[1]
    rc = types["compact"](args, _vector(start, "paged_compact start", i32, n_seq, dev), path.data_ptr(),
                          path.stride(0) if n_seq > 1 else width, _vector(count, "paged_compact count", i32, n_seq, dev), width,
                          types["stream"](dev))
    if rc:
        check(rc, "paged_compact")


def paged_copy(pool, src, dst, scale=None):
    """neko_op_paged_copy: in every plane of pool (as in paged_compact), page dst[i] becomes a copy of page src[i] (int32)."""
    types = _types or _setup()
    args, _, dev = _planes(pool, scale, None, "paged_copy", types)
    n = src.numel()
    rc = types["copy"](args, _vector(src, "paged_copy src", types["i32"], n, dev), _vector(dst, "paged_copy dst", types["i32"], n, dev), n,
                       types["stream"](dev))
    if rc:
        check(rc, "paged_copy")


def sample_rows(logits, u=None, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """neko_op_sample_rows: a token for each row of logits [rows][vocab] (float32, float16, bfloat16; any row stride; unchanged)
    from u float64 [rows] in [0, 1) (None: greedy). temperature, top_k, top_p and min_p are numbers or tensors [rows] (float32,
    top_k int32). Returns token int32 [rows] (-1: nothing to take) and prob float32 [rows], the one with which it was taken."""
    import torch
    types = _types or _setup()
    dev = _on_device(logits, "sample_rows", types)
    if logits.dim() != 2 or (logits.shape[1] > 1 and logits.stride(1) != 1):
        raise NekoError("sample_rows: logits are [rows][vocab], the vocabulary contiguous")
    (rows, vocab), is_tensor, each, one = logits.shape, torch.is_tensor, [], []
    for v, what, dt in ((temperature, "temperature", "f32"), (top_p, "top_p", "f32"), (min_p, "min_p", "f32"), (top_k, "top_k", "i32")):
        each.append(_vector(v, "sample_rows " + what, types[dt], rows, dev) if is_tensor(v) else 0)
        one.append(0 if is_tensor(v) else v)
    token, prob = logits.new_empty(rows, dtype=types["i32"]), logits.new_empty(rows, dtype=types["f32"])
    if u is None and not each[0] and one[0] > 0:
        raise NekoError("sample_rows: a positive temperature needs the rows' numbers u")
    args = _SAMPLE.pack(logits.data_ptr(), _vector(u, "sample_rows u", types["f64"], rows, dev), *each, token.data_ptr(), prob.data_ptr(),
                        logits.stride(0) if rows > 1 else vocab, types.get(logits.dtype, -1), rows, vocab, max(-1, min(int(one[3]), 0x7fffffff)),
                        *(max(-3e38, min(x, 3e38)) if x == x else x for x in one[:3]), 0)
    rc = types["sample"](args, types["stream"](dev))
    if rc:
        check(rc, "sample_rows")
    return token, prob


def status():
    """neko_op_status: waits for the current stream and raises when a paged_append or paged_attention since the last call
    had a sequence with more new tokens than max_new, rows that are not there, or positions past the rotation table."""
    check(lib().neko_op_status(_stream()), "paged operators")


def trim(keep_bytes=0):
    """neko_op_trim: gives the operators' idle scratch memory on the current device back, beyond keep_bytes. Work that used it
    has to be synchronised with."""
    check(lib().neko_op_trim(keep_bytes), "trim")
