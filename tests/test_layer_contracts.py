"""What the decoder-layer operators and the model around them accept, refuse and
promise, as far as that needs no GPU."""

import math
import os
import shutil
import subprocess
from decimal import Decimal, localcontext

import pytest

from qwen3_engine_from_scratch_b200 import rope
from qwen3_engine_from_scratch_b200.rope import RotaryPlan, rotary_frequencies

TINY = dict(layers=1, hidden=32, heads=1, kv_heads=1, head_dim=16, intermediate=32, vocab=64, max_pos=8)


def test_model_refuses_plans_that_its_rotation_cannot_follow():
    """The fused QK-norm prologue pairs i with i + head_dim / 2: tables of another
    layout have the same shape and would turn q and k by the wrong angles."""
    from qwen3_engine_from_scratch_b200.e2e_model import Qwen3DecodeModel
    for plan in (RotaryPlan(16, layout="interleaved", device="cpu"), RotaryPlan(8, device="cpu")):
        with pytest.raises(AssertionError, match="rope_plan"):
            Qwen3DecodeModel("cpu", rope_plan=plan, **TINY)
        assert Qwen3DecodeModel("cpu", rope_plan=plan, qk_norm=False, **TINY).plan is plan
    with pytest.raises(AssertionError, match="rope_plan"):
        Qwen3DecodeModel("cpu", rope_plan=RotaryPlan(18, device="cpu"), qk_norm=False, **TINY)
    whole = RotaryPlan(16, device="cpu")
    assert Qwen3DecodeModel("cpu", rope_plan=whole, **TINY).plan is whole


def test_yarn_ramp_ends_beyond_the_last_pair_where_that_pair_still_turns():
    """The ramp over the pair's index ends at the first whole index at which a pair
    makes slow_turns or fewer, also where that lies past the last pair: written here
    for one pair at a time, in turns."""
    for rotary_dim, base, trained in ((128, 1e4, 131072), (64, 1e4, 131072), (128, 1e4, 65536), (26, 1e4, 32768),
                                      (8, 1e4, 32768), (128, 1e6, 32768), (16, 1e6, 8192), (64, 5e5, 8192)):
        factor, slow, fast = 4.0, 1.0, 32.0
        turns = lambda i: trained * base ** (-2.0 * i / rotary_dim) / (2 * math.pi)  # noqa: E731
        first, last = 0, 0
        while turns(first + 1) >= fast:              # the last whole index with fast_turns or more
            first += 1
        while turns(last) > slow:                    # the first with slow_turns or fewer
            last += 1
        got, _ = rotary_frequencies(rotary_dim, base=base, scaling="yarn", factor=factor, original_len=trained,
                                    slow_turns=slow, fast_turns=fast)
        for i, f in enumerate(got):
            squeezed = min(1.0, max(0.0, (i - first) / (last - first)))
            plain = base ** (-2.0 * i / rotary_dim)
            want = (1 - squeezed) * plain + squeezed * plain / factor
            assert f == pytest.approx(want, rel=1e-12), (rotary_dim, base, trained, i)
        # no pair that turns more than slow_turns is squeezed by the whole factor
        assert all(f > 1.0001 * base ** (-2.0 * i / rotary_dim) / factor
                   for i, f in enumerate(got) if turns(i) > slow)


def test_norms_refuse_a_missing_weight():
    """Not taken for a quantisation without a norm, which the C entry has for itself."""
    import torch
    from qwen3_engine_from_scratch_b200 import ops
    x = torch.ones(2, 16, dtype=torch.bfloat16)
    for norm in (ops.rms_norm, ops.rms_norm_fp8):
        with pytest.raises(AssertionError, match="weight"):
            norm(x, None)


def test_overlap_of_a_tensor_with_itself():
    import torch
    from qwen3_engine_from_scratch_b200 import ops
    t = torch.zeros(4, 6, 16)
    for fine in (t, t.transpose(0, 1), t[:, ::2], t[:, :, 3:9], t[:1].expand(1, 6, 16), t[:0], t[1:2, 3:4],
                 t[0].unflatten(0, (2, 3)).transpose(0, 2), t.as_strided((1, 6, 16), (0, 16, 1))):
        assert not ops._overlaps_itself(fine), (fine.shape, fine.stride())
    for bad in (t[:1].expand(4, 6, 16), t[:, :1].expand(4, 6, 16), t.as_strided((4, 6, 16), (90, 16, 1)),
                t.as_strided((4, 6, 16), (96, 15, 1)), t.as_strided((2, 4, 16), (24, 16, 1))):
        assert ops._overlaps_itself(bad), (bad.shape, bad.stride())


def test_c_entries_refuse_sizes_whose_indexes_would_pass_31_bits(native_lib):
    """Element, token and head indexes are 32-bit and step past the end by a block's
    share before the loops stop: sizes that close to 2^31 are refused, before a launch."""
    lib, fake, top = native_lib, 16, 2 ** 31 - 1
    norm = lambda hidden, weight: lib.b200_rms_norm(  # noqa: E731
        fake, hidden, None, 0, weight, fake, hidden, None if weight else fake, None, 0, 1, hidden, 1e-6, None, None)
    for hidden in (top, top - 7, top - 8191):
        assert norm(hidden, fake) == -1 and norm(hidden, None) == -1, hidden
    product = lambda m: lib.b200_linear(  # noqa: E731
        fake, 8, None, fake, 8, None, None, None, 0, fake, 8, m, 8, 8, 0, 0, 0, None, None)
    for m in (top, top - 1, top - 254):
        assert product(m) == -1, m
    rotary = lambda heads, kv, dim: lib.b200_rotary(  # noqa: E731
        fake, 8, 8, 8, fake, 8, 8, 8, fake, 8, 8, 8, fake, 8, 8, 8, fake, 0, 1, 0, fake, 1.0, 1, 1, heads, kv, dim, 8,
        0, None)
    for heads, kv, dim in ((top, 1, 8), (top, 0, 8), (1, top - 512, 8), (2 ** 30, 2 ** 30, 8), (1, 1, top),
                           (1, 1, top - 254)):
        assert rotary(heads, kv, dim) == -1, (heads, kv, dim)


ONCE = r"""
#include <cstdio>
#include <thread>
#include <vector>
#include "once.cuh"

static b200host::OncePerDevice once;
static int calls[64], value[64][4];   // plain data behind the flag, as the products' occupancies

int main() {
  int failures = 0;
  if (once.run(3, [] { return -5; }) != -5) ++failures;      // a failure is not kept
  for (int device = 0; device < 64; ++device) {
    std::vector<std::thread> threads;
    std::vector<int> seen(8);
    for (int t = 0; t < 8; ++t)
      threads.emplace_back([&, t] {
        if (once.run(device, [&] { ++calls[device]; for (int& v : value[device]) v = device + 1; return 0; }) == 0)
          seen[t] = value[device][t % 4];
      });
    for (auto& t : threads) t.join();
    for (int v : seen) failures += v != device + 1;
    failures += calls[device] != 1;
  }
  return failures != 0;
}
"""


def test_first_calls_from_several_threads(tmp_path):
    """One thread does a device's first-call work, the others see all of it; under the
    thread sanitizer, which exits with 66 where it finds a race."""
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("no g++")
    csrc = os.path.join(os.path.dirname(rope.__file__), "csrc")

    def run(source):
        (tmp_path / "t.cc").write_text(source)
        exe = str(tmp_path / "t")
        built = subprocess.run([gxx, "-std=c++17", "-O1", "-g", "-fsanitize=thread", "-I", csrc,
                                str(tmp_path / "t.cc"), "-o", exe], capture_output=True, text=True)
        if built.returncode:
            return None, built.stderr
        done = subprocess.run([exe], capture_output=True, text=True, timeout=120)
        return done.returncode, done.stderr

    if run("int main() { return 0; }")[0] != 0:
        pytest.skip("the thread sanitizer does not run here")
    code, text = run(ONCE)
    assert code == 0, text[-3000:]
    # linear.cu keeps its occupancies behind it, and no flag of its own
    with open(os.path.join(csrc, "linear.cu")) as f:
        source = f.read()
    assert "OncePerDevice" in source and "g_attr_done" not in source


PI = Decimal("3.14159265358979323846264338327950288419716939937510582097494459230781640628620899862803")


def turns_a_position(rotary_dim, base, factor=1):
    """rotary_dim / 2 exact turns a position (to 50 digits), f_i / factor."""
    with localcontext() as c:
        c.prec = 60
        return [(Decimal(base) ** (Decimal(-2 * i) / rotary_dim)) / factor / (2 * PI) for i in range(rotary_dim // 2)]


@pytest.mark.parametrize("rotary_dim,base", [(128, 1000000), (64, 10000), (6, 100), (256, 500000)])
def test_fractions_of_a_turn_against_50_digits(rotary_dim, base):
    """The plan's float64 frequencies leave 2^-54 of a turn a position: pow's and the
    exponent's rounding, 1.4 x 2^-53 of f <= 1, and 2 pi's and the quotient's, 1.4 more,
    all over 2 pi."""
    for factor in (1, 4):
        more = dict(scaling="linear", factor=float(factor)) if factor > 1 else {}
        plan = RotaryPlan(rotary_dim, base=float(base), device="cpu", **more)
        for got, want in zip(plan.turns.tolist(), turns_a_position(rotary_dim, base, factor)):
            with localcontext() as c:
                c.prec = 60
                off = abs(Decimal(got % 2 ** 64) / 2 ** 64 - want)
            assert off < Decimal(2) ** -54
