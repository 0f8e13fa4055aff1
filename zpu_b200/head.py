"""A language model's output head on the device (zpucuda_layer_norm,
zpucuda_distill_*, zpucuda_int8_* and zpucuda_sample).

The operators around the output projection: layer norm and its gradient, the
distillation loss from a teacher's top logits and its gradient, the linear
layer in 8-bit integers, and the choice of the next token.  Activations and
logits are [rows, n] CUDA tensors of float32, float16 or bfloat16, contiguous
along the row and with any row pitch (a slice of a wider tensor is read in
place); results are new tensors unless `out` names one.  With `stream`, the
call runs on that torch stream and its new tensors belong to it.
"""
import functools

from . import CUDA_STREAM_LEGACY, _capi
from ._capi import check, lib


@functools.cache
def _torch():
    import torch
    return torch


@functools.cache
def _codes():
    torch = _torch()
    return {torch.float32: _capi.F32, torch.float16: 2, torch.bfloat16: _capi.DT_BF16}


def _stream(x):
    """The current stream, a cudaStream_t, for a call on x.  A launch goes to
    the current device, so x has to be there.  (The handle without a Stream
    object around it: a call on one token is the shorter by 2 us.)"""
    C = _torch()._C
    dev = x.get_device()
    if dev != C._cuda_getDevice():
        _refuse(12, "the tensors are on %s, the current device is cuda:%d" % (x.device, C._cuda_getDevice()))
    # torch's default stream is the legacy NULL stream; NULL means the thread's
    # own stream to the C ABI, so it is named as cudaStreamLegacy.
    return C._cuda_getCurrentRawStream(dev) or CUDA_STREAM_LEGACY


def _refuse(status, text):
    raise _capi.ZpuCudaError(status, text)


def _code(name, t):
    code = _codes().get(t.dtype)
    if code is None:
        _refuse(9, "%s: dtype %s is not float32, float16 or bfloat16" % (name, t.dtype))
    return code


def _matrix(name, t, like=None, shape=None):
    """Checks a [rows, n] argument; its row pitch in elements."""
    size = t.shape
    if len(size) != 2:
        _refuse(5, "%s: %d axes, [rows, n] is wanted" % (name, len(size)))
    if shape is not None and size != shape:
        _refuse(2, "%s: shape %s, %s is wanted" % (name, tuple(size), tuple(shape)))
    _device(name, t, like)
    ld, step = t.stride()
    rows, n = size
    if step != 1 and n > 1:
        _refuse(7, "%s: its rows are not contiguous" % name)
    if rows <= 1:  # torch leaves the stride of an axis of one (or no) row arbitrary
        return n
    if ld < n:
        _refuse(7, "%s: its rows overlap" % name)
    return ld


def _device(name, t, like=None):
    if not t.is_cuda or (like is not None and t.get_device() != like.get_device()):
        _refuse(12, "%s is on %s" % (name, t.device if like is None or not t.is_cuda
                                     else "%s, not %s" % (t.device, like.device)))


def _vector(name, t, n, like, dtype=None):
    """Checks an optional [n] argument; its address."""
    if t is None:
        return None
    if t.dim() != 1 or t.numel() != n:
        _refuse(2, "%s: shape %s, (%d,) is wanted" % (name, tuple(t.shape), n))
    if dtype is not None and t.dtype != dtype:
        _refuse(3, "%s: dtype %s, %s is wanted" % (name, t.dtype, dtype))
    if not t.is_cuda or t.get_device() != like.get_device():
        _device(name, t, like)
    if n > 1 and not t.is_contiguous():
        _refuse(7, "%s is not contiguous" % name)
    return t.data_ptr()


def _output(name, out, like, shape=None, dtype=None):
    """`out`, checked, or a new tensor; and its row pitch."""
    if out is None and shape is None and dtype is None and like.is_contiguous():
        return _torch().empty_like(like), like.shape[1]
    if shape is None:
        shape = like.shape
    if dtype is None:
        dtype = like.dtype
    if out is None:
        return _torch().empty(shape, dtype=dtype, device=like.device), shape[1]
    if out.dtype != dtype:
        _refuse(3, "%s: dtype %s, %s is wanted" % (name, out.dtype, dtype))
    return out, _matrix(name, out, like, shape)


# ------------------------------------------------------------- layer norm
def _weights(x, gamma, beta):
    cols = x.shape[1]
    if gamma is not None and beta is not None and gamma.dtype != beta.dtype:
        _refuse(3, "gamma is %s, beta is %s" % (gamma.dtype, beta.dtype))
    g, b = _vector("gamma", gamma, cols, x), _vector("beta", beta, cols, x)
    some = gamma if gamma is not None else beta
    return (_capi.F32 if some is None else _code("gamma / beta", some)), g, b


def layer_norm(x, gamma=None, beta=None, eps=1e-5, out=None, stats=False, stream=None):
    """(x - mean) / sqrt(var + eps) * gamma + beta over each row of x.  With
    `stats` also the rows' mean and 1 / sqrt(var + eps) (float32), which
    layer_norm_grad takes.  `out` may be x."""
    if stream is not None:
        with _torch().cuda.stream(stream):
            return layer_norm(x, gamma, beta, eps, out, stats)
    torch = _torch()
    ldx, code = _matrix("x", x), _code("x", x)
    wt, g, b = _weights(x, gamma, beta)
    rows, cols = x.shape
    y, ldy = _output("out", out, x)
    if stats:
        mean = torch.empty(rows, dtype=torch.float32, device=x.device)
        rstd = torch.empty_like(mean)
    check(lib().zpucuda_layer_norm(code, x.data_ptr(), ldx, wt, g, b, y.data_ptr(), ldy,
                                   mean.data_ptr() if stats else None, rstd.data_ptr() if stats else None,
                                   rows, cols, eps, _stream(x)))
    return (y, mean, rstd) if stats else y


def layer_norm_grad(dy, x, mean, rstd, gamma=None, out=None, stream=None):
    """(dx, dgamma, dbeta) of layer_norm for the output's gradient dy: dx like
    x (in `out`, which may be dy or x), dgamma and dbeta like gamma (float32
    without one)."""
    if stream is not None:
        with _torch().cuda.stream(stream):
            return layer_norm_grad(dy, x, mean, rstd, gamma, out)
    torch = _torch()
    ldx, code = _matrix("x", x), _code("x", x)
    if dy.dtype != x.dtype:
        _refuse(3, "dy is %s, x is %s" % (dy.dtype, x.dtype))
    lddy = _matrix("dy", dy, x, x.shape)
    rows, cols = x.shape
    m = _vector("mean", mean, rows, x, torch.float32)
    r = _vector("rstd", rstd, rows, x, torch.float32)
    wt, g, _ = _weights(x, gamma, None)
    dx, lddx = _output("out", out, x)
    dgamma = torch.empty(cols, dtype=gamma.dtype if gamma is not None else torch.float32, device=x.device)
    dbeta = torch.empty_like(dgamma)
    work = torch.empty(lib().zpucuda_layer_norm_grad_work(rows, cols), dtype=torch.uint8, device=x.device)
    check(lib().zpucuda_layer_norm_grad(code, dy.data_ptr(), lddy, x.data_ptr(), ldx, m, r, wt, g, dx.data_ptr(), lddx,
                                        dgamma.data_ptr(), dbeta.data_ptr(), rows, cols, work.data_ptr(), work.numel(),
                                        _stream(x)))
    return dx, dgamma, dbeta


# ------------------------------------------------------------- distillation
def _distill_args(logits, teacher, indices, weight):
    torch = _torch()
    ld, code = _matrix("logits", logits), _code("logits", logits)
    rows, vocab = logits.shape
    if teacher.dim() != 2 or teacher.shape[0] != rows:
        _refuse(2, "teacher: shape %s, [%d, top] is wanted" % (tuple(teacher.shape), rows))
    if indices.dtype not in (torch.int32, torch.int64):
        _refuse(9, "indices: dtype %s is not int32 or int64" % indices.dtype)
    ldt = _matrix("teacher", teacher, logits)
    ldi = _matrix("indices", indices, logits, teacher.shape)
    w = _vector("weight", weight, rows, logits, torch.float32)
    head = (code, logits.data_ptr(), ld, _code("teacher", teacher), teacher.data_ptr(), ldt,
            4 if indices.dtype == torch.int32 else _capi.DT_I64, indices.data_ptr(), ldi, w)
    return head, (rows, vocab, teacher.shape[1])


def distill_loss(logits, teacher, indices, temperature=1.0, weight=None, stream=None):
    """(loss, lse): weight * T^2 * KL(teacher's listed softmax || student's
    softmax) of each row at temperature T, and log sum exp(logits / T).
    teacher: the teacher's top logits [rows, top] at the vocabulary `indices`
    (int32 / int64; -1: no entry).  A row with weight 0 or no entry gives 0."""
    if stream is not None:
        with _torch().cuda.stream(stream):
            return distill_loss(logits, teacher, indices, temperature, weight)
    torch = _torch()
    head, dims = _distill_args(logits, teacher, indices, weight)
    loss = torch.empty(dims[0], dtype=torch.float32, device=logits.device)
    lse = torch.empty_like(loss)
    check(lib().zpucuda_distill_loss(*head, temperature, loss.data_ptr(), lse.data_ptr(), *dims,
                                     _stream(logits)))
    return loss, lse


def distill_grad(logits, teacher, indices, lse, dloss=None, temperature=1.0, weight=None, out=None, stream=None):
    """The gradient of sum(dloss * loss) with regard to the logits, from
    distill_loss's lse.  `out` may be the logits."""
    if stream is not None:
        with _torch().cuda.stream(stream):
            return distill_grad(logits, teacher, indices, lse, dloss, temperature, weight, out)
    torch = _torch()
    head, dims = _distill_args(logits, teacher, indices, weight)
    l = _vector("lse", lse, dims[0], logits, torch.float32)
    d = _vector("dloss", dloss, dims[0], logits, torch.float32)
    g, ldg = _output("out", out, logits)
    check(lib().zpucuda_distill_grad(*head, temperature, l, d, g.data_ptr(), ldg, *dims,
                                     _stream(logits)))
    return g


def distill_value_and_grad(logits, teacher, indices, dloss=None, temperature=1.0, weight=None, out=None, stream=None):
    """(loss, dlogits): distill_loss and distill_grad from one reading of the
    logits.  `out` may be the logits."""
    if stream is not None:
        with _torch().cuda.stream(stream):
            return distill_value_and_grad(logits, teacher, indices, dloss, temperature, weight, out)
    torch = _torch()
    head, dims = _distill_args(logits, teacher, indices, weight)
    d = _vector("dloss", dloss, dims[0], logits, torch.float32)
    loss = torch.empty(dims[0], dtype=torch.float32, device=logits.device)
    g, ldg = _output("out", out, logits)
    check(lib().zpucuda_distill_value_and_grad(*head, temperature, d, loss.data_ptr(), g.data_ptr(), ldg, *dims,
                                               _stream(logits)))
    return loss, g


# ------------------------------------------------------------- 8-bit integers
def quantize_rows(x, stream=None):
    """(q, scale): int8 rows and their float32 scales, scale = max |row| / 127."""
    if stream is not None:
        with _torch().cuda.stream(stream):
            return quantize_rows(x)
    torch = _torch()
    ldx, code = _matrix("x", x), _code("x", x)
    rows, cols = x.shape
    # a row pitch of a multiple of 16 bytes, as the product reads best
    q = torch.empty((rows, (cols + 15) // 16 * 16), dtype=torch.int8, device=x.device)[:, :cols]
    scale = torch.empty(rows, dtype=torch.float32, device=x.device)
    check(lib().zpucuda_int8_quantize(code, x.data_ptr(), ldx, q.data_ptr(), _matrix("q", q), scale.data_ptr(),
                                      rows, cols, _stream(x)))
    return q, scale


def _int8(name, t, like=None):
    if t.dtype != _torch().int8:
        _refuse(3, "%s: dtype %s, int8 is wanted" % (name, t.dtype))
    return _matrix(name, t, like)


def int8_matmul(a, a_scale, b, b_scale, bias=None, dtype=None, out=None, stream=None):
    """(a @ b.T) * a_scale[:, None] * b_scale + bias for int8 a [m, k] and b
    [n, k] with float32 scales per row, summed exactly; float32 unless `dtype`
    or `out` says otherwise."""
    if stream is not None:
        with _torch().cuda.stream(stream):
            return int8_matmul(a, a_scale, b, b_scale, bias, dtype, out)
    torch = _torch()
    lda, ldb = _int8("a", a), _int8("b", b, a)
    m, k = a.shape
    n = b.shape[0]
    if b.shape[1] != k:
        _refuse(2, "a is %s, b is %s" % (tuple(a.shape), tuple(b.shape)))
    sa = _vector("a_scale", a_scale, m, a, torch.float32)
    sb = _vector("b_scale", b_scale, n, a, torch.float32)
    bi = _vector("bias", bias, n, a, torch.float32)
    if dtype is None:
        dtype = out.dtype if out is not None else torch.float32
    y, ldy = _output("out", out, a, (m, n), dtype)
    check(lib().zpucuda_int8_matmul(a.data_ptr(), lda, sa, b.data_ptr(), ldb, sb, bi, _code("out", y), y.data_ptr(),
                                    ldy, m, n, k, _stream(a)))
    return y


class Int8Linear:
    """y = x @ weight.T + bias with int8 weights [cols, inner] and a float32
    scale per output channel, x quantised by row as it comes.  Made from
    quantised weights, or by Int8Linear.from_float.  Weights at a row pitch of
    a multiple of 16 bytes are kept as they are, others copied to one.  `out`
    may be x.  The tensors that a layer has been made with are its own for
    good (their values may change); others are another layer."""

    weight = property(lambda self: self._weight)
    scale = property(lambda self: self._scale)
    bias = property(lambda self: self._bias)

    def __init__(self, weight, scale, bias=None):
        torch = _torch()
        _int8("weight", weight)
        cols, inner = weight.shape
        if _vector("scale", scale, cols, weight, torch.float32) is None:
            _refuse(16, "scale: a tensor of (%d,) is wanted" % cols)
        _vector("bias", bias, cols, weight, torch.float32)
        self._ld = weight.stride(0) if cols > 1 else (inner + 15) // 16 * 16
        if self._ld % 16 or weight.data_ptr() % 16:
            self._ld = (inner + 15) // 16 * 16
            kept = torch.empty((cols, self._ld), dtype=torch.int8, device=weight.device)[:, :inner]
            weight = kept.copy_(weight)
        self._weight, self._scale, self._bias = weight, scale, bias

    @classmethod
    def from_float(cls, weight, bias=None, stream=None):
        """From float32 / float16 / bfloat16 weights [cols, inner]."""
        if stream is not None:
            with _torch().cuda.stream(stream):
                return cls.from_float(weight, bias)
        return cls(*quantize_rows(weight), bias)

    def __call__(self, x, out=None, stream=None):
        if stream is not None:
            with _torch().cuda.stream(stream):
                return self(x, out)
        torch = _torch()
        weight, bias = self._weight, self._bias
        ldx, code = _matrix("x", x, weight), _code("x", x)
        rows, inner = x.shape
        cols = weight.shape[0]
        if inner != weight.shape[1]:
            _refuse(2, "x is %s, the weight %s" % (tuple(x.shape), tuple(weight.shape)))
        y, ldy = _output("out", out, x, (rows, cols))
        work = torch.empty(lib().zpucuda_int8_linear_work(rows, inner), dtype=torch.uint8, device=x.device)
        check(lib().zpucuda_int8_linear(code, x.data_ptr(), ldx, weight.data_ptr(), self._ld,
                                        self._scale.data_ptr(), None if bias is None else bias.data_ptr(),
                                        y.data_ptr(), ldy, rows, cols, inner, work.data_ptr(), work.numel(),
                                        _stream(x)))
        return y


# ------------------------------------------------------------- the next token
def sample(logits, uniform, temperature=None, top_k=None, top_p=None, min_p=None, stream=None):
    """(token, logprob): a token (int64) of each row of logits, drawn with the
    given uniform numbers (float32 / float64 in [0, 1)), and its log
    probability among the tokens kept.  temperature (float32; <= 0: the
    likeliest token), top_k (int32; <= 0: all), top_p (float32; >= 1: all) and
    min_p (float32; <= 0: all) are [rows] tensors, or plain numbers for every
    row.  NaN and -inf logits are never drawn; a row of nothing else gives -1."""
    if stream is not None:
        with _torch().cuda.stream(stream):
            return sample(logits, uniform, temperature, top_k, top_p, min_p)
    torch = _torch()
    ld, code = _matrix("logits", logits), _code("logits", logits)
    rows, vocab = logits.shape
    if uniform.dtype not in (torch.float32, torch.float64):
        _refuse(9, "uniform: dtype %s is not float32 or float64" % uniform.dtype)
    u = _vector("uniform", uniform, rows, logits)
    keep = []

    def each(name, v, dtype):
        if v is None:
            return None
        if not hasattr(v, "data_ptr"):
            v = torch.full((rows,), v, dtype=dtype, device=logits.device)
            keep.append(v)
        return _vector(name, v, rows, logits, dtype)

    rules = (each("temperature", temperature, torch.float32), each("top_k", top_k, torch.int32),
             each("top_p", top_p, torch.float32), each("min_p", min_p, torch.float32))
    token = torch.empty(rows, dtype=torch.int64, device=logits.device)
    logprob = torch.empty(rows, dtype=torch.float32, device=logits.device)
    check(lib().zpucuda_sample(code, logits.data_ptr(), ld, 0 if uniform.dtype == torch.float64 else 1, u, *rules,
                               token.data_ptr(), logprob.data_ptr(), rows, vocab, _stream(logits)))
    return token, logprob
