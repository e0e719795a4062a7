"""Plans of the classifier head's loss, without a GPU: scratch sizes, what is refused, documentation that compiles."""
import ctypes

import pytest

import cudnntest_b200 as cb


def _bytes(plan, grad):
    return cb.lib().wino_xent_workspace_bytes(ctypes.byref(plan.desc), grad)


@pytest.mark.parametrize("n,d,v,kw", [
    (677, 9184, 1383, dict(label_smoothing=0.1, scratch_limit=16 << 20)),         # dz counts against the limit with gradients alone
    (1457, 1, 7119, dict()),                                                      # plain kernels without gradients alone
    (14201, 1, 393, dict(scratch_limit=16 << 20, bias=True)),
    (58, 5, 4892, dict(scratch_limit=1, dtype="fp32x3")),
    (64, 4096, 1000, dict()), (1, 1, 1, dict()), (0, 8, 8, dict()), (4096, 1024, 32000, dict(dtype="fp32x3")),
])
def test_a_plan_with_gradients_has_room_for_forward(n, d, v, kw):
    """`forward` may be called on it: its scratch is at least that of either call."""
    plan = cb.LinearXent(n, d, v, device="meta", **kw)
    need = max(_bytes(plan, 0), _bytes(plan, 1))
    assert plan.ws_bytes >= need and plan.workspace.numel() >= need
    alone = cb.LinearXent(n, d, v, device="meta", grad=False, **kw)
    assert alone.ws_bytes == _bytes(alone, 0)


def _round(a, q):
    return -(-a // q) * q


def _desc(n, d, v, dtype, limit, **kw):
    s = cb.XentDesc()
    s.n, s.d, s.v, s.dtype, s.scratch_limit = n, d, v, dtype, limit
    for k, x in kw.items():
        setattr(s, k, x)
    return s


@pytest.mark.parametrize("dtype", [cb.BF16, cb.FP32X3])
@pytest.mark.parametrize("smoothing", [0.0, 0.1])
@pytest.mark.parametrize("limit", [1, 1000, 1 << 14, 1 << 20, 16 << 20, 1 << 28])
def test_scratch_of_the_loss_alone_stays_within_the_limit(dtype, smoothing, limit):
    """Beside scratch_limit: the statistics, five vectors over the rows, x and W repacked, and 256 bytes of rounding for each."""
    L = cb.lib()
    planes = 1 if dtype == cb.BF16 else 3
    for n in (1, 8, 64, 128, 1000, 4096, 16384, 100000):
        for d in (1, 9, 64, 2050, 1 << 14, 1 << 20):
            for v in (1, 15, 128, 1000, 8192, 30000):
                s = _desc(n, d, v, dtype, limit, label_smoothing=smoothing)
                stats = -(-v // 128) * n * (8 if smoothing == 0 else 12)
                packed = (n + v) * _round(d, 8) * 2 * planes
                assert L.wino_xent_workspace_bytes(ctypes.byref(s), 0) <= limit + stats + 20 * n + packed + 12 * 256, (n, d, v)


@pytest.mark.parametrize("n,d,v,dtype", [(4096, 1024, 9000, cb.BF16), (8192, 2048, 20000, cb.BF16), (4096, 256, 9000, cb.FP32X3), (2304, 1024, 2050, cb.BF16)])
def test_column_sums_of_kept_logits_count_against_the_limit(n, d, v, dtype):
    """Float logits (unsplit here: more tiles than CTA pairs), dz and the column sums for dbias are kept only where all three fit:
    runs of 32 rows each behind 8192 classes, up to then at least one run per SM."""
    L = cb.lib()
    planes = 1 if dtype == cb.BF16 else 3
    z, dz = n * _round(v, 4) * 4, n * _round(v, 8) * 2 * planes
    sums = (-(-n // 32) if v > 8192 else 148) * _round(v, 8) * 4

    def at(limit):
        return L.wino_xent_workspace_bytes(ctypes.byref(_desc(n, d, v, dtype, limit, has_bias=1)), 1)
    kept = at(1 << 60)
    assert kept >= z + dz + sums
    assert at(z + dz + sums - 1) < kept
    no_bias = _desc(n, d, v, dtype, z + dz, has_bias=0)
    if dtype == cb.FP32X3:                                        # without a bias there are no such sums
        assert L.wino_xent_workspace_bytes(ctypes.byref(no_bias), 1) >= z + dz


@pytest.mark.parametrize("dtype", [cb.BF16, cb.FP32X3])
def test_small_gradients_keep_to_the_limit_or_to_a_piece(dtype):
    """The plain kernels' logits, parts and column sums: within the limit, or what a piece of 256 classes of dz takes."""
    L = cb.lib()
    planes = 1 if dtype == cb.BF16 else 3
    for n, d, v in ((128, 16, 64), (128, 1, 128), (1, 1 << 20, 15), (2, 1 << 18, 31), (7, 1 << 16, 33), (128, 1000, 128), (1, 1, 1)):
        for limit in (1, 1 << 12, 1 << 15, 1 << 30):
            for bias in (0, 1):
                s = _desc(n, d, v, dtype, limit, has_bias=bias)
                floor = n * 256 * 2 * planes + (-(-n // 32)) * 256 * 4 * bias
                dx = 64 * (n + 256) * _round(d, 4) * 4             # at most 64 float parts of dx, and of 256 classes of dW
                packed = (n + v) * _round(d, 8) * 2 * planes
                got = L.wino_xent_workspace_bytes(ctypes.byref(s), 1)
                assert got <= max(limit, floor) + -(-v // 128) * n * 8 + 20 * n + 14 * 256 + (0 if limit == 1 << 30 else packed + dx), (n, d, v, limit, bias)


def test_scratch_is_kept_for_the_stream_that_uses_it(monkeypatch):
    """A call on another stream than the plan's own tells the allocator, so that a plan dropped while the call runs does not hand
    its scratch to somebody else."""
    import torch
    from cudnntest_b200 import head
    plan = cb.LinearXent(8, 16, 10, device="meta")
    told, now = [], [5]

    class Scratch:
        def data_ptr(self):
            return 1 << 20

        def record_stream(self, stream):
            told.append(stream)
    monkeypatch.setattr(head, "_raw_stream", lambda index: now[0])
    monkeypatch.setattr(head, "_call", lambda *args: None)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda index=None: now[0])
    monkeypatch.setattr(plan, "_inputs", lambda *args: (0, 0, None, 0))
    plan.workspace, plan._index, plan._made_on = Scratch(), 0, 5
    x, w = torch.empty(8, 16, dtype=torch.bfloat16, device="meta"), torch.empty(10, 16, dtype=torch.bfloat16, device="meta")
    for call in (lambda: plan.forward(x, w, None), lambda: plan.loss_and_grad(x, w, None, need_dx=False, need_dw=False)):
        told.clear()
        now[0] = 5
        call()
        assert told == []
        now[0] = 6
        call()
        assert told == [6]


@pytest.mark.parametrize("kw", [dict(n=2 ** 32 + 8), dict(n=2 ** 31), dict(d=2 ** 32 + 16), dict(v=2 ** 32 + 10), dict(v=-2 ** 32 + 10), dict(reduction=2 ** 32),
                                dict(ignore_index=2 ** 64 + 3), dict(ignore_index=2 ** 63), dict(ldx=2 ** 64 + 16), dict(scratch_limit=2 ** 64)])
def test_numbers_that_the_descriptor_cannot_hold(kw):
    """They are refused: taken modulo 2^32 or 2^64 they would be another plan for tensors of these sizes."""
    with pytest.raises(ValueError):
        cb.LinearXent(**{**dict(n=8, d=16, v=10, device="meta"), **kw})
    plan = cb.LinearXent(8, 16, 10, device="meta", ignore_index=-2 ** 63)
    assert plan.desc.ignore_index == -2 ** 63


def test_handed_in_scratch_is_contiguous():
    """A tensor whose elements share memory has less of it than it has elements."""
    import torch
    plan = cb.LinearXent(8, 16, 10, device="meta")
    for strided in (torch.empty(1, dtype=torch.uint8, device="meta").expand(plan.ws_bytes), torch.empty(2 * plan.ws_bytes, dtype=torch.uint8, device="meta")[::2]):
        with pytest.raises(ValueError):
            cb.LinearXent(8, 16, 10, device="meta", workspace=strided)
    own = torch.empty(plan.ws_bytes // 4 + 1, dtype=torch.float32, device="meta")
    assert cb.LinearXent(8, 16, 10, device="meta", workspace=own).workspace is own
    small = torch.empty(8, dtype=torch.uint8, device="meta")
    assert cb.LinearXent(8, 16, 10, device="meta", workspace=small).workspace is not small


def test_classifier_head_takes_images_first():
    """Features whose first axis is not the batch (a CHWN stack's output) would be flattened across images."""
    import torch
    from cudnntest_b200 import vgg
    head_ = vgg.ClassifierHead(6, 4 * 2 * 2, 10, device="meta")
    for shape in ((6, 16), (6, 2, 2, 4), (6, 4, 2, 2)):
        assert head_._flat(torch.empty(shape, dtype=torch.bfloat16, device="meta")).shape == (6, 16)
    for shape in ((4, 2, 2, 6), (16, 6), (96,), (6, 15), (7, 16), (6, 2, 2, 5), (2, 3, 16), ()):
        with pytest.raises(ValueError):
            head_._flat(torch.empty(shape, dtype=torch.bfloat16, device="meta"))


def test_classifier_head_of_no_images():
    import torch
    from cudnntest_b200 import vgg
    head_ = vgg.ClassifierHead(0, 16, 10, device="meta")
    assert head_._flat(torch.empty((0, 2, 2, 4), dtype=torch.bfloat16, device="meta")).shape == (0, 16)
    with pytest.raises(ValueError):
        head_._flat(torch.empty((0, 2, 2, 5), dtype=torch.bfloat16, device="meta"))


def test_classifier_head_keeps_what_it_owns_for_the_stream(monkeypatch):
    import torch
    from cudnntest_b200 import head, vgg
    head_ = vgg.ClassifierHead(6, 16, 10, device="meta")
    x, t = torch.empty((6, 16), dtype=torch.bfloat16, device="meta"), torch.empty(6, dtype=torch.int64, device="meta")
    for call in (head_.loss, head_.loss_and_grad):                # no GPU: refused
        with pytest.raises(ValueError):
            call(x, t)
    head_.plan._index = 0
    told = []
    monkeypatch.setattr(head, "_raw_stream", lambda index: 6)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda index=None: 6)
    monkeypatch.setattr(torch.Tensor, "record_stream", lambda self, stream: told.append(id(self)))
    owned = {id(head_.weight), id(head_.bias)}
    for call, want in ((head_.loss, owned), (head_.loss_and_grad, owned | {id(head_._step)})):
        told.clear()
        with pytest.raises(ValueError):
            call(x, t)
        assert want <= set(told)


def test_classifier_head_takes_features_inside_wider_rows():
    """loss took only contiguous ones, loss_and_grad any pitch."""
    import torch
    from cudnntest_b200 import vgg
    head_ = vgg.ClassifierHead(6, 16, 10, device="meta")
    for x in (torch.empty((6, 24), dtype=torch.bfloat16, device="meta")[:, :16], torch.empty((16, 6), dtype=torch.bfloat16, device="meta").t(),
              torch.empty((6, 2, 2, 8), dtype=torch.bfloat16, device="meta")[..., :4]):
        assert head_._flat(x).is_contiguous() and head_._flat(x).shape == (6, 16)


def test_the_documented_c_example_compiles(tmp_path):
    """INTEGRATION.md's calls, with every tensor declared as what the text says it is (device memory: pointers)."""
    import os
    import re
    import shutil
    import subprocess
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    cc = shutil.which("gcc")
    if cc is None:
        pytest.skip("no C compiler")
    text = open(os.path.join(root, "INTEGRATION.md")).read()
    code = re.search(r"## 5\..*?```c\n(.*?)```", text, re.S).group(1)
    (tmp_path / "example.c").write_text('#include <stddef.h>\n#include "wino.h"\n'
                                        "void example(int images, int classes, unsigned long long seed, unsigned long long step, void* features, void* h,\n"
                                        "             void* dh, void* dfeatures, void* weight, void* dweight, float* bias, float* dbias, float* loss,\n"
                                        "             long long* labels, void* workspace, wino_stream_t stream) {\n" + code + "(void)bytes;\n}\n")
    r = subprocess.run([cc, "-std=c11", "-Wall", "-Werror", "-fsyntax-only", "-I", os.path.join(root, "include"), "example.c"], cwd=tmp_path,
                       capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stderr


_TURNS = r"""
#include <cstdio>
#include <vector>
#include "xent_turns.cuh"
using namespace wino;
int main() {
    for (unsigned most : {1u, 2u, 7u, 74u})
        for (unsigned u0 = 1; u0 <= 3 * most + 2; ++u0)
            for (unsigned u1 = 0; u1 <= 3 * most + 2; ++u1)
                for (double ratio : {1.0, 1.4, 2.0, 5.0}) {
                    const unsigned total = u0 + u1, pairs = total < most ? total : most, lead = xe_turns_lead(u0, u1, pairs, ratio);
                    std::vector<int> seen(total, 0);
                    unsigned fewest = ~0u, longest = 0;
                    for (unsigned p = 0; p < pairs; ++p) {
                        const XeTurns t(u0, u1, pairs, lead, p);
                        unsigned i = 0;
                        long long last = -1;
                        for (long long u; (u = t.at(i)) >= 0; ++i, last = u)
                            if (u >= total || u <= last || seen[u]++) return printf("unit %lld of %u + %u on %u pairs\n", u, u0, u1, pairs), 1;
                        if (t.at(i + 1) >= 0 || t.at(i + 1000) >= 0) return printf("a unit behind the last\n"), 1;
                        if (i < fewest) fewest = i;
                        if (i > longest) longest = i;
                    }
                    for (int s : seen)
                        if (!s) return printf("a unit of %u + %u is missing\n", u0, u1), 1;
                    /* nobody waits while another has two units to do */
                    if (fewest == 0 || (total <= most && longest > 1)) return printf("%u + %u units on %u pairs: %u ... %u\n", u0, u1, pairs, fewest, longest), 1;
                    /* without units taken ahead the shares differ by one at most */
                    if (!lead && longest > fewest + 1) return printf("%u + %u units on %u pairs: %u ... %u\n", u0, u1, pairs, fewest, longest), 1;
                }
    return 0;
}
"""


def test_two_products_share_the_pairs(tmp_path):
    """Every unit of both products exactly once, in order, and no pair idle while another has two."""
    import os
    import shutil
    import subprocess
    cxx = shutil.which("g++")
    if cxx is None:
        pytest.skip("no C++ compiler")
    csrc = os.path.join(os.path.dirname(cb.__file__), "csrc")
    (tmp_path / "turns.cpp").write_text(_TURNS)
    r = subprocess.run([cxx, "-std=c++17", "-O2", "-Wall", "-Werror", "-I", csrc, "turns.cpp", "-o", "turns"], cwd=tmp_path, capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stderr
    r = subprocess.run(["./turns"], cwd=tmp_path, capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stdout


def test_measured_sizes_split_inside_the_products():
    """Gradients of more than 64 rows or classes, on the side that was measured faster: split beforehand, the longer matrix alone takes
    six bytes an element of scratch."""
    for n, d, v, inside in ((8000, 2048, 128, True), (128, 2048, 20000, True), (4000, 2048, 128, False), (128, 512, 20000, False)):
        got = cb.LinearXent(n, d, v, dtype="fp32x3", bias=True, device="meta")
        assert (_bytes(got, 1) < max(n, v) * d * 6) == inside, (n, d, v)


def test_wait_codes_name_their_kernel():
    """A wait that ran out reports a code that one kernel alone uses."""
    import glob
    import os
    import re
    csrc = os.path.join(os.path.dirname(cb.__file__), "csrc")
    values = {}
    for path in glob.glob(os.path.join(csrc, "xent*.cu*")):
        values.update((name, int(code)) for name, code in re.findall(r"(X[ET]_WAIT_\w+) = (\d+)", open(path).read()))
    used = {}
    for name in ("xent_gemm.cu", "xent_thin.cu"):
        used[name] = {values[code] for code in re.findall(r"X[ET]_WAIT_\w+", open(os.path.join(csrc, name)).read())}
        assert len(used[name]) == 4
    assert not used["xent_gemm.cu"] & used["xent_thin.cu"]
