"""The vocabulary losses without a device: the oracle's gradient against differences, and refusals."""
import ctypes as C
import os
import re

import pytest

torch = pytest.importorskip("torch")

import loss_oracle as ref
import thiran_b200 as thb
from thiran_b200 import losses

BIG = 1 << 40  # an address that nothing reads


def test_oracle_gradient_is_the_difference_quotient():
    g = torch.Generator().manual_seed(1)
    z = torch.randn((4, 11), generator=g, dtype=torch.float64)
    ids = torch.tensor([[3, 3, 7], [0, -1, 10], [-1, -1, -1], [5, 6, 2]])
    lists = ref.teacher_lists(ids, torch.randn((4, 3), generator=g), 1.5)
    slope = ref.losses(z, lists)[2]
    step = 1e-5
    for t in range(4):
        for v in range(11):
            d = torch.zeros_like(z)
            d[t, v] = step
            quotient = (ref.losses(z + d, lists)[0] - ref.losses(z - d, lists)[0]).sum() / (2 * step)
            assert abs(float(quotient - slope[t, v])) < 1e-8  # step^2 / 6 and 2^-52 * 4 / step


def test_oracle_agrees_with_torch():
    g = torch.Generator().manual_seed(2)
    z = torch.randn((5, 9), generator=g, dtype=torch.float64)
    labels = torch.tensor([0, 8, -100, 3, 3])
    loss, _, _, _ = ref.losses(z, ref.label_lists(labels, 9))
    assert torch.allclose(loss, torch.nn.functional.cross_entropy(z, labels, reduction="none"))
    ids = torch.stack([torch.randperm(9, generator=g)[:4] for _ in range(5)])
    s = torch.randn((5, 4), generator=g, dtype=torch.float64)
    q = torch.zeros_like(z).scatter_(1, ids, torch.softmax(s / 2, 1))
    divergence = torch.nn.functional.kl_div(torch.log_softmax(z / 2, 1), q, reduction="none").sum(1)
    assert torch.allclose(ref.losses(z / 2, ref.teacher_lists(ids, s, 2.0))[0], divergence)


def test_spreads_tell_how_sums_are_made():
    """Sums of 1024 products keep the bound on lse; sums of the whole width and logits in bf16 do not.
    Slopes of two summands keep the tighter bound on gradients, slopes of one only the wider."""
    g = torch.Generator().manual_seed(3)
    h, w, at = ref.well_known(24, 300, 4096, g, "cpu")
    z = h.double() @ w.double().T
    want = torch.logsumexp(z, 1)
    assert ref.spread(torch.logsumexp(ref.cut_sums(h, w, 1024).double(), 1), want)[0] < ref.LSE_SPREAD
    assert ref.spread(torch.logsumexp(ref.cut_sums(h, w, 4096).double(), 1), want)[0] > ref.LSE_SPREAD
    assert ref.spread(torch.logsumexp(z.bfloat16().double(), 1), want)[0] > ref.LSE_SPREAD
    h, w = torch.randn((48, 256), generator=g).bfloat16(), (torch.randn((500, 256), generator=g) / 8).bfloat16()
    slope = ref.losses(h.double() @ w.double().T, ref.label_lists(torch.randint(0, 500, (48,), generator=g), 500))[2]
    slope = slope * torch.rand((48, 1), generator=g)
    first = slope.bfloat16().double()
    second = first + (slope - first).bfloat16().double()
    for rounded, tight in ((first, False), (second, True)):
        for a, b, x in ((slope, rounded, w.double()), (slope.T, rounded.T, h.double())):
            off = ref.spread((b @ x).bfloat16(), a @ x)[1]
            assert off < ref.GRADIENT_SPREAD[tight] and (tight or off > ref.GRADIENT_SPREAD[True])


def linear_desc(**changes):
    d = losses.LinearLossDesc(rows=16, vocab=64, dim=32, hidden=BIG, ld_hidden=32, weight=2 * BIG, ld_weight=32,
                              labels=3 * BIG, ignore_index=-100, entries=0, scale=1.0, loss=4 * BIG, lse=5 * BIG,
                              grad_loss=6 * BIG, grad_hidden=7 * BIG, ld_grad_hidden=32, grad_weight=8 * BIG,
                              ld_grad_weight=32, workspace=9 * BIG, workspace_bytes=1 << 30)
    for k, v in changes.items():
        setattr(d, k, v)
    return d


def distill_desc(**changes):
    d = losses.DistillDesc(rows=16, vocab=64, logits=BIG, ld_logits=64, dtype=thb.F32, teacher_ids=2 * BIG,
                           teacher_logits=3 * BIG, teacher_dtype=thb.F32, entries=4, scale=1.0, loss=4 * BIG,
                           lse=5 * BIG, grad_loss=6 * BIG, grad_logits=7 * BIG, ld_grad_logits=64)
    for k, v in changes.items():
        setattr(d, k, v)
    return d


def refused(name, desc, code="GPU-LOSS-ARGUMENT", says=""):
    """Arguments are checked before the device is looked for, so this needs none."""
    fail = C.create_string_buffer(1024)
    status = getattr(thb.lib(), name)(0, C.byref(desc) if desc is not None else None, None, fail, len(fail))
    text = fail.value.decode()
    assert status == thb.STATUS_ABI and text.startswith(code) and says in text, text


FORWARD, BACKWARD = "thb_linear_loss_forward", "thb_linear_loss_backward"
TEACHER = dict(labels=None, teacher_ids=10 * BIG, teacher_logits=11 * BIG, teacher_dtype=thb.F32, entries=4)


@pytest.mark.parametrize("changes,says", [
    (dict(vocab=0), "vocab"), (dict(dim=0), "dim"), (dict(rows=1 << 31), "2^30"), (dict(scale=0.0), "scale"),
    (dict(scale=-1.0), "scale"), (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale"), (dict(scale=2.0 ** 101), "scale"),
    (dict(scale=2.0 ** -101), "scale"),
    (dict(hidden=None), "hidden is null"), (dict(hidden=BIG + 1), "hidden is not aligned"), (dict(ld_hidden=31), "hidden"),
    (dict(weight=None), "weight is null"), (dict(ld_weight=31), "weight"), (dict(labels=BIG + 4096 + 4), "labels is not"),
    (dict(labels=None), "entries"), (dict(teacher_ids=10 * BIG), "both"),
    (dict(TEACHER, entries=1025), "1024"), (dict(TEACHER, entries=0), "1024"),
    (dict(TEACHER, teacher_dtype=thb.I64), "teacher logits"), (dict(TEACHER, teacher_ids=None), "teacher_ids is null"),
    (dict(TEACHER, teacher_logits=None), "teacher_logits is null"),
    (dict(workspace=None), "workspace"), (dict(workspace=9 * BIG + 128), "256"),
])
def test_linear_refusals(changes, says):
    refused(FORWARD, linear_desc(**changes), says=says)
    refused(BACKWARD, linear_desc(**changes), says=says)


@pytest.mark.parametrize("name,changes,says", [
    (FORWARD, dict(loss=None), "loss is null"), (FORWARD, dict(lse=None), "lse is null"),
    (FORWARD, dict(loss=5 * BIG + 60), "loss overlaps lse"), (FORWARD, dict(lse=BIG + 64), "lse overlaps hidden"),
    (FORWARD, dict(workspace=BIG - 256), "workspace overlaps hidden"),
    (BACKWARD, dict(grad_loss=None), "grad_loss is null"), (BACKWARD, dict(grad_hidden=None), "grad_hidden is null"),
    (BACKWARD, dict(grad_weight=None), "grad_weight is null"), (BACKWARD, dict(ld_grad_weight=31), "grad_weight"),
    (BACKWARD, dict(grad_hidden=BIG), "grad_hidden overlaps hidden"),
    (BACKWARD, dict(grad_weight=2 * BIG + 4094), "grad_weight overlaps weight"),
    (BACKWARD, dict(grad_weight=7 * BIG), "grad_weight overlaps grad_hidden"),
])
def test_linear_output_refusals(name, changes, says):
    refused(name, linear_desc(**changes), says=says)


@pytest.mark.parametrize("name", ["thb_distill_forward", "thb_distill_backward"])
@pytest.mark.parametrize("changes,says", [
    (dict(vocab=0), "vocab"), (dict(vocab=(1 << 30) + 1, ld_logits=1 << 31), "vocab exceeds"), (dict(rows=1 << 28), "rows"),
    (dict(dtype=thb.I64), "logits must be"), (dict(scale=0.0), "scale"), (dict(entries=0), "1024"),
    (dict(entries=1025), "1024"), (dict(logits=None), "logits is null"), (dict(logits=BIG + 2), "aligned"),
    (dict(ld_logits=63), "logits"), (dict(teacher_dtype=0), "teacher logits"), (dict(teacher_ids=None), "teacher_ids"),
    (dict(grad_loss=None), "grad_loss is null"), (dict(lse=None), "lse is null"), (dict(ld_grad_logits=63), "grad_logits"),
    (dict(grad_logits=BIG + 4), "grad_logits overlaps logits"),
    (dict(grad_logits=BIG, ld_grad_logits=65), "grad_logits overlaps logits"),
    (dict(grad_logits=2 * BIG), "grad_logits overlaps teacher_ids"),
])
def test_distill_refusals(name, changes, says):
    refused(name, distill_desc(**changes), says=says)


def test_more_refusals():
    for name in (FORWARD, BACKWARD, "thb_distill_forward", "thb_distill_backward"):
        refused(name, None, says="null")
    refused("thb_distill_forward", distill_desc(grad_logits=None), says="without grad_logits")
    refused("thb_distill_backward", distill_desc(grad_logits=None), says="grad_logits is null")
    refused("thb_distill_forward", distill_desc(loss=BIG), says="loss overlaps logits")
    refused(FORWARD, linear_desc(ld_weight=1 << 62), "GPU-SIZE-OVERFLOW")


def side_by_side(columns, pitch):
    """Slices of one buffer, `columns` bf16 apart, for hidden states and weights of width 32, and
    f32 for logits of width 64."""
    return (linear_desc(ld_hidden=pitch, ld_grad_hidden=pitch, grad_hidden=BIG + 2 * columns),
            linear_desc(ld_weight=pitch, ld_grad_weight=pitch, grad_weight=2 * BIG + 2 * columns),
            distill_desc(ld_logits=2 * pitch, ld_grad_logits=2 * pitch, grad_logits=BIG + 8 * columns))


@pytest.mark.parametrize("columns,pitch", [(31, 64), (33, 64), (32, 63), (40, 71), (1, 64), (63, 64), (0, 64)])
def test_slices_that_share_elements_are_refused(columns, pitch):
    hidden, weight, logits = side_by_side(columns, pitch)
    refused(BACKWARD, hidden, says="grad_hidden overlaps hidden")
    refused(BACKWARD, weight, says="grad_weight overlaps weight")
    if columns:  # (0: in place)
        for name in ("thb_distill_forward", "thb_distill_backward"):
            refused(name, logits, says="grad_logits overlaps logits")


def test_a_single_row_steps_nowhere():
    far = 1 << 63
    refused(BACKWARD, linear_desc(rows=1, ld_hidden=far, ld_grad_hidden=far, grad_hidden=BIG + 2), says="overlaps hidden")


@pytest.mark.skipif(torch.cuda.is_available(), reason="the addresses are nobody's")
@pytest.mark.parametrize("columns,pitch", [(32, 64), (32, 65), (40, 72), (64 + 32, 64), (5 * 64 + 32, 64)])
def test_slices_side_by_side_are_taken(columns, pitch):
    """Arguments pass, and the device is what is missing."""
    hidden, weight, logits = side_by_side(columns, pitch)
    fail = C.create_string_buffer(1024)
    for name, desc in ((BACKWARD, hidden), (BACKWARD, weight), ("thb_distill_forward", logits),
                       ("thb_distill_backward", logits)):
        assert getattr(thb.lib(), name)(0, C.byref(desc), None, fail, len(fail)) == thb.STATUS_BACKEND, fail.value


def test_binding_refuses_wrong_tensors():
    """Types, shapes and devices are checked by the binding (CPU tensors are no CUDA tensors)."""
    h, w = torch.zeros((4, 8), dtype=torch.bfloat16), torch.zeros((16, 8), dtype=torch.bfloat16)
    loss, lse = torch.zeros(4), torch.zeros(4)
    with pytest.raises(thb.GpuError, match="CUDA device") as err:
        thb.linear_cross_entropy(h, w, torch.zeros(4, dtype=torch.int64), loss, lse, torch.zeros(8))
    assert err.value.code == "GPU-LOSS-ARGUMENT" and err.value.status == thb.STATUS_ABI
    with pytest.raises(thb.GpuError, match="CUDA device"):
        thb.distillation(torch.zeros((4, 16)), torch.zeros((4, 2), dtype=torch.int64), torch.zeros((4, 2)), loss, lse)
    with pytest.raises(thb.GpuError, match="temperature"):
        losses._temperature(0.0)
    cpu = -1  # the ordinal of CPU tensors
    for t, says in ((torch.zeros((4, 9)), "shape"), (torch.zeros((4, 8), dtype=torch.float64), "float64"),
                    (torch.zeros((8, 4)).T, "contiguous"), (torch.zeros(8).expand(4, 8), "overlapping")):
        with pytest.raises(thb.GpuError, match=says):
            losses._matrix("x", t, 4, 8, torch.float32, cpu)
    for t, says in ((torch.zeros(5), "shape"), (torch.zeros(8)[::2], "contiguous"), (torch.zeros(4).double(), "float64")):
        with pytest.raises(thb.GpuError, match=says):
            losses._vector("x", t, 4, torch.float32, cpu)


def test_descriptor_layouts():
    """The binding's structures have the header's sizes (tests of the fields run on a device)."""
    assert C.sizeof(losses.LinearLossDesc) == 184 and C.sizeof(losses.DistillDesc) == 120


@pytest.mark.skipif(torch.cuda.is_available(), reason="checks the no-device path")
def test_no_device_no_fallback():
    fail = C.create_string_buffer(1024)
    for name, desc in ((FORWARD, linear_desc()), (BACKWARD, linear_desc()), ("thb_distill_forward", distill_desc()),
                       ("thb_distill_backward", distill_desc())):
        assert getattr(thb.lib(), name)(0, C.byref(desc), None, fail, len(fail)) == thb.STATUS_BACKEND
        assert fail.value.decode().startswith("GPU-DRIVER-NOT-FOUND")


def test_linear_losses_issue_tcgen05_and_tma():
    source = os.path.join(os.path.dirname(losses.__file__), "csrc")
    kernels, helpers = (open(os.path.join(source, name)).read() for name in ("linear_loss.cu", "tensor_core.cuh"))
    assert "tcgen05.mma" in helpers and "cp.async.bulk.tensor" in helpers and "tcgen05.ld" in helpers
    for call in ("mmaPair(", "mma(", "tmaLoad2dPair(", "tmaLoad2d(", "tmemFetch32("):
        assert call in kernels and call in helpers
    for legacy in ("wgmma", "mma.sync", "wmma::"):
        assert legacy not in kernels + helpers


def test_what_is_remembered_of_a_device_is_remembered_by_device():
    """Function-local statics of the host code are tables by device, or hold nothing of a device."""
    source = os.path.join(os.path.dirname(losses.__file__), "csrc")
    for name in ("linear_loss.cu", "distill.cu"):
        text = open(os.path.join(source, name)).read()
        held = re.findall(r"^ +static (?!constexpr|__device__)(.*)$", text, re.M)
        assert held
        for line in held:
            assert re.match(r"std::mutex mutex;|std::map<std::tuple<.*, int, .*known;|std::atomic<uint64_t> ready\{0\};|"
                            r"std::atomic<uint32_t> pairs\[kKnownDevices\]\{\};|const uint32_t spins = ", line), (name, line)


def test_copies_in_flight_are_waited_for_behind_the_last_role():
    """Any role's wait may run out after the copies' own role has left, so their wait stands behind
    the barrier at which all roles have ended."""
    source = os.path.join(os.path.dirname(losses.__file__), "csrc")
    for name, end, drains in (("distill.cu", "\n    __syncthreads();\n    if (threadIdx.x == 0 && abortFlag)", ["drained &= mbarWait("]),
                              ("linear_loss.cu", "\n    __syncthreads();\n    if (threadIdx.x == 0 && abortFlag)",
                               ["!landed<G::stages>(full, issuedHere, issuedByPeer", "!landed<G::stages>(full, issuedHere, issuedHere"])):
        text = open(os.path.join(source, name)).read()
        assert text.count(end) == 1
        for drain in drains:
            assert text.count(drain) == 1 and text.index(drain) > text.index(end), (name, drain)


def test_no_wait_is_a_mere_sleep():
    """What is in flight is counted, not given a while."""
    source = os.path.join(os.path.dirname(losses.__file__), "csrc")
    for name in ("linear_loss.cu", "linear_score.cuh", "distill.cu"):
        assert "nanosleep" not in open(os.path.join(source, name)).read()
