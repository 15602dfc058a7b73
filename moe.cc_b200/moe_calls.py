"""moe_calls.py — the Python calls of a decode step (kv_plan, qk_norm_rope,
paged_attention, route) through ctypes: what moe_cuda.py offers where the
CPython extension (py/moe_fast.c) was not built, for want of Python's headers.
Arguments, checks and errors are the extension's; a call takes the host 9 to 20
us instead of 4 to 13. torch is imported with the first call."""
import ctypes as C

import moe_cuda as mc

I32, F32 = "torch.int32", "torch.float32"
ELEM = {"torch.float32": mc.F32, "torch.float16": mc.F16, "torch.bfloat16": mc.BF16}
SCORES = {"softmax": 0, "sigmoid": 1}
INT_MAX = 2**31 - 1


def _refuse(msg, code=mc.MOE_ERR_INVALID):
    raise mc.MoeError(code, msg)


def _tensor(t, what):
    import torch
    if not isinstance(t, torch.Tensor) or t.dim() > 4:
        _refuse(f"{what}: a tensor of at most 4 dimensions is wanted")
    return t


def _flat(t, dtype, n, dev, what):
    """Address of a contiguous tensor of n elements of one type on cuda:dev; None: None."""
    if t is None:
        return None
    _tensor(t, what)
    if str(t.dtype) != dtype or t.numel() != n or t.get_device() != dev or not t.is_contiguous():
        _refuse(f"{what}: a contiguous tensor of {n} elements of {dtype} on cuda:{dev} is wanted")
    return t.data_ptr()


def _heads(t, what, rows, heads, hd, dtype, dev):
    """(address, row stride) of [rows][heads][hd] whose rows may lie apart."""
    s = _tensor(t, what).stride()
    if tuple(t.shape) != (rows, heads, hd) or t.get_device() != dev or t.dtype != dtype or \
            (rows and ((s[2] != 1 and hd > 1) or (s[1] != hd and heads > 1))):
        _refuse(f"{what}: [{rows}][{heads}][{hd}] of {dtype} on cuda:{dev} with contiguous rows is wanted")
    return t.data_ptr(), s[0] if rows > 1 else heads * hd


def _cache(k, v):
    _tensor(k, "k_cache")
    _tensor(v, "v_cache")
    if not k.is_cuda or k.get_device() != v.get_device() or k.dim() != 4 or max(k.shape) > INT_MAX:
        _refuse("kv cache: [n_pages][page_size][n_kv][head_dim] on a CUDA device is wanted")
    return mc.kv_cache(k, v), k.get_device(), k.dtype


def _int(v, what):
    try:
        v = v.__index__()
    except (AttributeError, TypeError):
        _refuse(f"{what}: a 32-bit integer is wanted")
    return v if -INT_MAX - 1 <= v <= INT_MAX else _refuse(f"{what}: a 32-bit integer is wanted")


def _real(v, what):
    try:
        return float(v)
    except (TypeError, ValueError):
        _refuse(f"{what}: a number is wanted")


def _stream(s):
    s = mc._stream(s)
    return s if s is None or isinstance(s, int) else _refuse("stream: a CUDA stream is wanted")


def kv_plan(past_len, new_len, page_size, n_pages, free_pages, block_table, row_seq, row_pos, row_slot, kv_len=None,
            free_head=None, free_head_out=None, status=None, stream=None):
    """kv_plan(past_len, new_len, page_size, n_pages, free_pages, block_table, row_seq, row_pos, row_slot, kv_len=None,
            free_head=None, free_head_out=None, status=None, stream=None)

    moe_kv_plan_dev on int32 tensors; past_len may be None (nothing held yet). block_table [sequences][pages]; the three
    row tensors of one length; free_head, free_head_out of one element, status of three."""
    _tensor(block_table, "block_table")
    if block_table.dim() != 2 or not block_table.is_cuda or max(block_table.shape) > INT_MAX:
        _refuse("block_table: [sequences][pages] on a CUDA device is wanted")
    (n, mp), dev = block_table.shape, block_table.get_device()
    cap, free = _tensor(row_seq, "row_seq").numel(), _tensor(free_pages, "free_pages").numel()
    if max(cap, free) > INT_MAX:
        _refuse("kv_plan: more than 2^31 - 1 rows or free pages", mc.MOE_ERR_UNSUPPORTED)
    mc.check(mc.lib().moe_kv_plan_dev(
        _flat(past_len, I32, n, dev, "past_len"), _flat(new_len, I32, n, dev, "new_len"), n, _int(page_size, "page_size"),
        _int(n_pages, "n_pages"), _flat(free_pages, I32, free, dev, "free_pages"), free, _flat(free_head, I32, 1, dev, "free_head"),
        _flat(block_table, I32, n * mp, dev, "block_table"), mp, _flat(kv_len, I32, n, dev, "kv_len"),
        _flat(row_seq, I32, cap, dev, "row_seq"), _flat(row_pos, I32, cap, dev, "row_pos"), _flat(row_slot, I32, cap, dev, "row_slot"),
        cap, _flat(free_head_out, I32, 1, dev, "free_head_out"), _flat(status, I32, 3, dev, "status"), _stream(stream)))


def qk_norm_rope(q, k, v, k_cache, v_cache, row_pos, row_slot, q_out, rope=None, q_norm=None, k_norm=None, eps=1e-6,
                 stream=None):
    """qk_norm_rope(q, k, v, k_cache, v_cache, row_pos, row_slot, q_out, rope=None, q_norm=None, k_norm=None, eps=1e-6,
                 stream=None)

    moe_qk_norm_rope_dev. q [rows][n_q][head_dim] (None: keys and values only), k, v [rows][n_kv][head_dim], rows of one
    stride each; rope [positions][rot_dim] fp32, the cosines then the sines; row_slot None: queries only (k, v are then
    not read and may be None)."""
    c, dev, ct = _cache(k_cache, v_cache)
    x = _tensor(k if q is None else q, "k" if q is None else "q")
    dt, hd = ELEM.get(str(x.dtype)), c.head_dim
    if dt is None or x.dim() != 3 or max(x.shape) > INT_MAX:
        _refuse("q, k: [rows][heads][head_dim] of float32, float16 or bfloat16 is wanted")
    rows, n_q, n_rope, rot = x.shape[0], 0, 0, 0
    qp = op = kp = vp = None
    ldq = ldo = ldk = ldv = 0
    if q is not None:
        n_q = q.shape[1]
        qp, ldq = _heads(q, "q", rows, n_q, hd, x.dtype, dev)
        op, ldo = _heads(q_out, "q_out", rows, n_q, hd, ct, dev)
    if row_slot is not None:
        kp, ldk = _heads(k, "k", rows, c.n_kv, hd, x.dtype, dev)
        vp, ldv = _heads(v, "v", rows, c.n_kv, hd, x.dtype, dev)
    if rope is not None:
        if _tensor(rope, "rope").dim() != 2 or max(rope.shape) > INT_MAX:
            _refuse("rope: [positions][rot_dim] is wanted")
        n_rope, rot = rope.shape
    mc.check(mc.lib().moe_qk_norm_rope_dev(
        qp, ldq, kp, ldk, vp, ldv, dt, rows, n_q, _flat(q_norm, F32, hd, dev, "q_norm"), _flat(k_norm, F32, hd, dev, "k_norm"),
        _real(eps, "eps"), _flat(rope, F32, n_rope * rot, dev, "rope"), rot, n_rope, _flat(row_pos, I32, rows, dev, "row_pos"),
        _flat(row_slot, I32, rows, dev, "row_slot"), op, ldo, C.byref(c), _stream(stream)))


def paged_attention(q, k_cache, v_cache, block_table, row_pos, out, workspace, max_kv, scale, lse=None, row_seq=None,
                    stream=None):
    """paged_attention(q, k_cache, v_cache, block_table, row_pos, out, workspace, max_kv, scale, lse=None, row_seq=None,
                    stream=None)

    moe_paged_attention_dev. q, out [rows][n_q][head_dim]; workspace: a contiguous tensor of any type (None where none is
    needed)."""
    c, dev, ct = _cache(k_cache, v_cache)
    if _tensor(q, "q").dim() != 3 or _tensor(block_table, "block_table").dim() != 2 or max(*q.shape, *block_table.shape) > INT_MAX:
        _refuse("q: [rows][heads][head_dim], block_table: [sequences][pages] are wanted")
    (rows, n_q, _), (n_seq, mp) = q.shape, block_table.shape
    qp, ldq = _heads(q, "q", rows, n_q, c.head_dim, ct, dev)
    op, ldo = _heads(out, "out", rows, n_q, c.head_dim, ct, dev)
    wp, wn = None, 0
    if workspace is not None:
        if _tensor(workspace, "workspace").get_device() != dev or not workspace.is_contiguous():
            _refuse(f"workspace: a contiguous tensor on cuda:{dev} is wanted")
        wp, wn = workspace.data_ptr(), workspace.nbytes
    mc.check(mc.lib().moe_paged_attention_dev(
        qp, ldq, C.byref(c), _flat(block_table, I32, n_seq * mp, dev, "block_table"), n_seq, mp,
        _flat(row_seq, I32, rows, dev, "row_seq"), _flat(row_pos, I32, rows, dev, "row_pos"), rows, n_q, _int(max_kv, "max_kv"),
        _real(scale, "scale"), op, ldo, _flat(lse, F32, rows * n_q, dev, "lse"), wp, wn, _stream(stream)))


def route(logits, topk_idx, topk_p, bias=None, score="softmax", groups=1, keep_groups=1, group_top=1, renorm=True,
          scale=1.0, stream=None):
    """route(logits, topk_idx, topk_p, bias=None, score='softmax', groups=1, keep_groups=1, group_top=1, renorm=True,
          scale=1.0, stream=None)

    moe_route_dev: topk_idx (int32) and topk_p (fp32) [rows][top_k] of logits [rows][experts] (rows may lie apart);
    score 'softmax' or 'sigmoid'."""
    _tensor(logits, "logits")
    _tensor(topk_idx, "topk_idx")
    dt, dev = ELEM.get(str(logits.dtype)), logits.get_device()
    if dt is None or logits.dim() != 2 or topk_idx.dim() != 2 or not logits.is_cuda or max(*logits.shape, topk_idx.shape[1]) > INT_MAX or \
            (logits.shape[0] and logits.shape[1] > 1 and logits.stride(1) != 1):
        _refuse("logits: [rows][experts] of float32, float16 or bfloat16 with contiguous experts on a CUDA device, "
                "topk_idx: [rows][top_k] are wanted")
    if score not in SCORES:
        _refuse("score: 'softmax' or 'sigmoid' is wanted")
    (rows, E), k = logits.shape, topk_idx.shape[1]
    mc.check(mc.lib().moe_route_dev(
        logits.data_ptr(), logits.stride(0) if rows > 1 else E, dt, rows, E, _flat(bias, F32, E, dev, "bias"), SCORES[score],
        _int(groups, "groups"), _int(keep_groups, "keep_groups"), _int(group_top, "group_top"), k, bool(renorm), _real(scale, "scale"),
        _flat(topk_idx, I32, rows * k, dev, "topk_idx"), _flat(topk_p, F32, rows * k, dev, "topk_p"), _stream(stream)))
