"""The language-model head's argument checks, which come before any CUDA call:
each bad argument is refused with its status and a message, here without a GPU."""
import pytest

F32, F16, BF16, I32, I64, F64 = 1, 2, 9, 4, 3, 0
A = 1 << 20  # an address that a refused call never reads
OUT_OF_SHAPE, NOT_SUPPORTED, INVALID = 5, 9, 16


@pytest.fixture(scope="module")
def L():
    from zpu_b200 import build
    build.build()
    from zpu_b200 import _capi
    return _capi.lib()


def call(L, name, order, good, **bad):
    args = dict(good, **bad)
    st = getattr(L, name)(*[args[k] for k in order.split()])
    return st, L.zpucuda_last_error().decode()


NORM = "dt x ldx wt gamma beta y ldy mean rstd rows cols eps stream"
NORM_OK = dict(dt=F32, x=A, ldx=8, wt=F32, gamma=A, beta=A, y=A, ldy=8, mean=A, rstd=A, rows=0, cols=8, eps=1e-5, stream=1)
NORM_GRAD = "dt dy lddy x ldx mean rstd wt gamma dx lddx dgamma dbeta rows cols work nwork stream"
NORM_GRAD_OK = dict(dt=F32, dy=A, lddy=8, x=A, ldx=8, mean=A, rstd=A, wt=F32, gamma=A, dx=A, lddx=8, dgamma=None,
                    dbeta=None, rows=0, cols=8, work=None, nwork=0, stream=1)
TEACH = "dt x ld tt teacher ldt it index ldi weight T "
TEACH_OK = dict(dt=F32, x=A, ld=8, tt=F32, teacher=A, ldt=4, it=I64, index=A, ldi=4, weight=None, T=2.0, loss=A, lse=A,
                dloss=None, d=A, ldd=8, rows=0, vocab=8, top=4, stream=1)
LOSS = TEACH + "loss lse rows vocab top stream"
GRAD = TEACH + "lse dloss d ldd rows vocab top stream"
BOTH = TEACH + "dloss loss d ldd rows vocab top stream"
QUANT = "dt x ldx q ldq scale rows cols stream"
QUANT_OK = dict(dt=F32, x=A, ldx=8, q=A, ldq=8, scale=A, rows=0, cols=8, stream=1)
MUL = "a lda sa b ldb sb bias dt out ldo m n k stream"
MUL_OK = dict(a=A, lda=8, sa=A, b=A, ldb=8, sb=A, bias=None, dt=F32, out=A, ldo=4, m=0, n=4, k=8, stream=1)
LINEAR = "dt x ldx w ldw sw bias y ldy rows cols inner work nwork stream"
LINEAR_OK = dict(dt=F32, x=A, ldx=8, w=A, ldw=8, sw=A, bias=None, y=A, ldy=4, rows=0, cols=4, inner=8, work=A, nwork=1 << 20,
                 stream=1)
SAMPLE = "dt x ld ut u temp k p mp token logprob rows vocab stream"
SAMPLE_OK = dict(dt=F32, x=A, ld=8, ut=F32, u=A, temp=None, k=None, p=None, mp=None, token=A, logprob=None, rows=0, vocab=8,
                 stream=1)

CASES = [
    ("zpucuda_layer_norm", NORM, NORM_OK, [
        (dict(dt=I32), NOT_SUPPORTED, "x: the type"), (dict(wt=I64), NOT_SUPPORTED, "gamma: the type"),
        (dict(ldx=7), OUT_OF_SHAPE, "x: the row pitch"), (dict(ldy=7), OUT_OF_SHAPE, "y: the row pitch"),
        (dict(rows=-1), OUT_OF_SHAPE, "rows"), (dict(cols=0), OUT_OF_SHAPE, "cols"),
        (dict(eps=-1.0), INVALID, "eps"), (dict(eps=float("nan")), INVALID, "eps"),
        (dict(rows=1, x=None), INVALID, "x: null"), (dict(rows=1, y=None), INVALID, "y: null"),
        (dict(x=A + 2), INVALID, "not aligned"), (dict(dt=BF16, y=A + 1), INVALID, "not aligned")]),
    ("zpucuda_layer_norm_grad", NORM_GRAD, NORM_GRAD_OK, [
        (dict(dt=F64), NOT_SUPPORTED, "dy: the type"), (dict(lddy=7), OUT_OF_SHAPE, "dy"),
        (dict(lddx=0), OUT_OF_SHAPE, "dx"), (dict(rows=1, mean=None), INVALID, "mean"),
        (dict(rows=1, rstd=None), INVALID, "rstd"), (dict(rows=1, x=None), INVALID, "x: null"),
        (dict(rows=1, dgamma=A), INVALID, "work"), (dict(rows=1, dgamma=A, work=A, nwork=63), INVALID, "work"),
        (dict(rows=1, dbeta=A, work=A + 4, nwork=1 << 20), INVALID, "work")]),
    ("zpucuda_distill_loss", LOSS, TEACH_OK, [
        (dict(T=0.0), INVALID, "temperature"), (dict(T=float("inf")), INVALID, "temperature"),
        (dict(T=float("nan")), INVALID, "temperature"), (dict(T=-1.0), INVALID, "temperature"),
        (dict(top=1025, ldt=1025, ldi=1025), NOT_SUPPORTED, "1024"), (dict(top=-1), OUT_OF_SHAPE, "top"),
        (dict(it=F32), NOT_SUPPORTED, "indices"), (dict(ldi=3), OUT_OF_SHAPE, "indices"),
        (dict(ldt=3), OUT_OF_SHAPE, "teacher"), (dict(vocab=0), OUT_OF_SHAPE, "vocab"),
        (dict(vocab=1 << 31, ld=1 << 31), NOT_SUPPORTED, "2^31"), (dict(rows=1, loss=None), INVALID, "loss"),
        (dict(rows=1, index=None), INVALID, "indices"), (dict(tt=I64), NOT_SUPPORTED, "teacher")]),
    ("zpucuda_distill_grad", GRAD, TEACH_OK, [
        (dict(rows=1, lse=None), INVALID, "lse"), (dict(ldd=7), OUT_OF_SHAPE, "dlogits"),
        (dict(rows=1, d=None), INVALID, "dlogits"), (dict(T=0.0), INVALID, "temperature")]),
    ("zpucuda_distill_value_and_grad", BOTH, TEACH_OK, [
        (dict(rows=1, loss=None), INVALID, "loss"), (dict(rows=1, d=None), INVALID, "dlogits"),
        (dict(ld=7), OUT_OF_SHAPE, "logits")]),
    ("zpucuda_int8_quantize", QUANT, QUANT_OK, [
        (dict(rows=-1), OUT_OF_SHAPE, "negative"), (dict(ldq=7), OUT_OF_SHAPE, "q"), (dict(dt=7), NOT_SUPPORTED, "x"),
        (dict(rows=1, q=None), INVALID, "q"), (dict(rows=1, scale=None), INVALID, "scale")]),
    ("zpucuda_int8_matmul", MUL, MUL_OK, [
        (dict(k=131072, lda=131072, ldb=131072), NOT_SUPPORTED, "32 bits"), (dict(lda=7), OUT_OF_SHAPE, "a"),
        (dict(ldb=7), OUT_OF_SHAPE, "b"), (dict(m=1, sa=None), INVALID, "a"), (dict(sb=None), INVALID, "b"),
        (dict(m=-1), OUT_OF_SHAPE, "negative"), (dict(ldo=3), OUT_OF_SHAPE, "out"), (dict(dt=I32), NOT_SUPPORTED, "out"),
        (dict(m=64 * 65535 + 1), NOT_SUPPORTED, "rows")]),
    ("zpucuda_int8_linear", LINEAR, LINEAR_OK, [
        (dict(rows=2, work=None), INVALID, "work"), (dict(rows=2, nwork=39), INVALID, "work"),
        (dict(rows=2, work=A + 8), INVALID, "work"), (dict(ldx=7), OUT_OF_SHAPE, "x"), (dict(ldw=7), OUT_OF_SHAPE, "b"),
        (dict(inner=-1), OUT_OF_SHAPE, "negative")]),
    ("zpucuda_sample", SAMPLE, SAMPLE_OK, [
        (dict(vocab=0), OUT_OF_SHAPE, "vocab"), (dict(vocab=(1 << 22) + 1, ld=1 << 23), NOT_SUPPORTED, "2^22"),
        (dict(ut=F16), NOT_SUPPORTED, "uniform"), (dict(rows=1, u=None), INVALID, "uniform"),
        (dict(rows=1, token=None), INVALID, "token"), (dict(dt=I64), NOT_SUPPORTED, "logits"),
        (dict(ld=7), OUT_OF_SHAPE, "logits")]),
]


@pytest.mark.parametrize("name,order,good,bad", CASES, ids=[c[0] for c in CASES])
def test_refusals(L, name, order, good, bad):
    for change, status, text in bad:
        st, msg = call(L, name, order, good, **change)
        assert st == status, (change, st, msg)
        assert text in msg, (change, msg)


@pytest.mark.parametrize("name,order,good", [c[:3] for c in CASES if c[0] != "zpucuda_layer_norm_grad"],
                         ids=[c[0] for c in CASES if c[0] != "zpucuda_layer_norm_grad"])
def test_no_rows_is_no_work(L, name, order, good):
    assert call(L, name, order, good)[0] == 0


def test_linear_workspace(L):
    assert L.zpucuda_int8_linear_work(0, 8) == 0
    assert L.zpucuda_int8_linear_work(3, 17) == 3 * 32 + 12
    assert L.zpucuda_int8_linear_work(-1, 8) == 0


def test_front_end_refuses_host_tensors():
    import torch
    import zpu_b200 as zc
    x = torch.zeros(2, 4)
    for f in (lambda: zc.layer_norm(x), lambda: zc.quantize_rows(x), lambda: zc.sample(x, torch.zeros(2)),
              lambda: zc.distill_loss(x, x, torch.zeros(2, 4, dtype=torch.int64))):
        with pytest.raises(zc.ZpuCudaError) as e:
            f()
        assert e.value.name == "DeviceMismatch"
    with pytest.raises(zc.ZpuCudaError) as e:
        zc.layer_norm(torch.zeros(3))
    assert e.value.name == "InvalidShape"


# ------------------------------------------------------------- sizes that the kernels go by, walked through on the host
def host(tmp_path, body, *flags):
    """The output of a C++ program about csrc/head_rules.h."""
    import os
    import subprocess
    from zpu_b200 import build
    src, exe = tmp_path / "rules.cpp", tmp_path / "rules"
    src.write_text('#include <stdio.h>\n#include <algorithm>\n#include "head_rules.h"\nusing namespace zc;\nint main() {\n%s\n}\n' % body)
    subprocess.run([os.environ.get("CXX", "g++"), "-std=c++17", "-O1", *flags, "-I", build.CSRC, str(src), "-o", str(exe)], check=True)
    return subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split()


def test_short_rows_are_read_inside_shared_memory(tmp_path):
    """The product of one or two tokens: the last byte that the last warp's last slot gives, over all sizes of a row, of a
    unit and of a block's share, lies inside what the kernel is launched with; and units of several rows do come up.
    (Four rows read whatever a unit has would end past it: 135168 bytes of 133120 at 2048 values by 8192 channels.)"""
    out = host(tmp_path, """
    long bad = 0, over = 0, several = 0, worst = 0;
    for (int k = 1; k <= 9000; k++)
        for (int per = 1; per <= 520; per++)
            for (int m = 1; m <= 2; m++) {
                const VecUnits U = vec_units(148l * per, k, 148);
                const long slot = GV_RING - GV_SLOT, smem = vec_smem(m, k);
                const int size = std::min(U.seg, k), last = (size + 15) / 16 * 16;  // lanes read 16 bytes that begin below size
                bad += U.rows < 1 || U.rows * U.seg > GV_SLOT || U.per > GV_CHANNELS || (U.segs > 1 && U.rows > 1);
                several += U.rows > 1;
                for (int rows = 1; rows <= U.rows; rows++) {  // the last unit of a round may have fewer
                    long end = 0, wide = 0;
                    for (int r = 0; r < rows; r += 4)
                        for (int i = 0; i < (U.rows == 1 ? 1 : 4); i++) {
                            end = std::max(end, slot + (long)vec_row(r + i, rows) * U.seg + last);
                            wide = std::max(wide, slot + (long)(r + i) * U.seg + last);
                        }
                    bad += end > GV_RING;
                    over += wide > smem;
                    if (k == 2048 && per == 56 && m == 1 && rows == 2) worst = wide;
                }
            }
    printf("%ld %d %d %ld", bad, several > 0, over > 0, worst);
    """)
    assert out == ["0", "1", "1", "135168"]


def test_weights_are_shifted_inside_their_bits(tmp_path):
    """floor(2^40 e) of every exponent of a 32-bit e in [0, 1] and of many significands, with no shift that C++ leaves open
    (the compiler's check ends the program at one)."""
    out = host(tmp_path, """
    long bad = 0;
    for (uint32_t u = 0; u <= 0x3f800000u; u += u % 0x800000u < 64 ? 1 : 4099) {
        const uint32_t exponent = u >> 23, significand = (u & 0x7fffffu) | (exponent ? 0x800000u : 0);
        const int up = (int)(exponent ? exponent : 1) - 150 + 40;  // e = significand * 2^(up - 40)
        const uint64_t want = up >= 0 ? (uint64_t)significand << up : up > -32 ? significand >> -up : 0;
        bad += weigh_bits(u) != want;
    }
    printf("%ld", bad);
    """, "-fsanitize=shift", "-fsanitize-undefined-trap-on-error")
    assert out == ["0"]


def test_rows_are_copied_from_inside_their_matrix(tmp_path):
    """Every row whose aligned 16 bytes begin before the matrix is known as such, over short rows, pitches and starts; it is
    not the first row alone."""
    out = host(tmp_path, """
    long bad = 0, others = 0;
    for (int n : {4, 8})  // elements of 16 bytes
        for (int base = 0; base < n; base++)
            for (int ld = 1; ld < 20; ld++)
                for (int row = 0; row < 40; row++) {
                    const int start = base + row * ld, skew = start % n;
                    const bool outside = start - skew < base;
                    bad += begins_outside((int64_t)row * ld, skew) != outside;
                    others += outside && row > 0;
                }
    printf("%ld %d", bad, others > 0);
    """)
    assert out == ["0", "1"]


VECTORS = [("zpucuda_layer_norm", NORM, NORM_OK, "mean rstd", 4), ("zpucuda_layer_norm_grad", NORM_GRAD, NORM_GRAD_OK, "mean rstd", 4),
           ("zpucuda_distill_loss", LOSS, TEACH_OK, "weight loss lse", 4), ("zpucuda_distill_loss", LOSS, TEACH_OK, "index", 8),
           ("zpucuda_distill_loss", LOSS, dict(TEACH_OK, it=I32), "index", 4),
           ("zpucuda_distill_grad", GRAD, TEACH_OK, "weight lse dloss", 4),
           ("zpucuda_distill_value_and_grad", BOTH, TEACH_OK, "weight dloss loss", 4),
           ("zpucuda_int8_quantize", QUANT, QUANT_OK, "scale", 4), ("zpucuda_int8_matmul", MUL, MUL_OK, "sa sb bias", 4),
           ("zpucuda_int8_linear", LINEAR, LINEAR_OK, "sw bias", 4), ("zpucuda_sample", SAMPLE, SAMPLE_OK, "u temp k p mp logprob", 4),
           ("zpucuda_sample", SAMPLE, dict(SAMPLE_OK, ut=F64), "u token", 8)]


@pytest.mark.parametrize("name,order,good,vectors,size", VECTORS, ids=["%s-%s" % (v[0], v[4]) for v in VECTORS])
def test_vectors_off_their_elements_are_refused(L, name, order, good, vectors, size):
    """An address that would fault on the GPU is refused by the call."""
    for v in vectors.split():
        for off in (1, size // 2):
            st, msg = call(L, name, order, good, **{v: A + off})
            assert st == INVALID and "not aligned" in msg, (v, off, st, msg)
        if name != "zpucuda_layer_norm_grad":
            assert call(L, name, order, good, **{v: A + size})[0] == 0


def test_any_number_of_rows_has_a_grid(tmp_path):
    """Up to the 2^31 - 1 rows that the distillation takes."""
    out = host(tmp_path, """
    long bad = 0;
    for (int64_t rows = 1; rows < 1ll << 31; rows += rows < 200000 ? 1 : rows < 2147000000ll ? 99991 : 1) {
        const RowGrid g = row_grid(rows);
        const int64_t over = (int64_t)g.y * g.z - rows;
        bad += g.y < 1 || g.y > 65535 || g.z < 1 || g.z > 65535 || over < 0 || over >= g.z;
    }
    printf("%ld", bad);
    """)
    assert out == ["0"]
