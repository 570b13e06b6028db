"""The operators of a bounded cache at their limits, on the host."""
import random
import re
import subprocess
import sys
from pathlib import Path

import pytest
import torch

from kinetics_b200 import EvictingKVManager, _lib, ops

CSRC = Path(__file__).resolve().parent.parent / "kinetics_b200" / "csrc"


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("kv_heads, heads", [(8, 32), (4, 32), (2, 4), (1, 8)])
@pytest.mark.parametrize("keep", [1000, 2000, 4000])
def test_a_managers_workspace_serves_every_number_of_active_slots(keep, kv_heads, heads, dtype):
    class Cfg:
        hidden_size, num_attention_heads, num_key_value_heads, head_dim, num_hidden_layers = 128 * heads, heads, kv_heads, 128, 1

    need = None
    for slots in (1, 8, 16, 24, 32, 64):
        kv = EvictingKVManager(Cfg, slots, 8192, "meta", dtype, keep=keep)
        need = need or [ops.decode_mass_workspace_bytes(n, kv_heads, heads // kv_heads, kv.pages_per_slot, dtype) for n in range(1, 65)]
        assert kv._decode_workspace().nbytes == max(need[:slots])


def test_a_size_for_fewer_sequences():
    size = lambda n, **kw: ops.decode_mass_workspace_bytes(n, 8, 4, 189, torch.bfloat16, **kw)
    assert size(16) == 0 < size(10)                                     # a cluster each; balanced
    assert size(16, fewer=True) == size(10) == size(10, fewer=True) and size(9, fewer=True) == 0
    assert size(0) == size(0, fewer=True) == 0


def test_a_decode_that_gives_up_waits_for_the_copies_of_all_lanes(tmp_path):
    """Lanes that issue in turn may stop anywhere; behind the barrier of the block each stage's last copy is waited for, by the stage's tag.
    Compiled here from the source, against a ring that is filled step by step."""
    text = (CSRC / "ktk_decode_mma.cu").read_text()
    rule = re.search(r"^__host__ __device__ constexpr int last_copy\(.*$", text, re.M).group(0)
    (tmp_path / "rule.cpp").write_text("#include <cstdio>\n#define __host__\n#define __device__\n" + rule + """
int main() { int tag, stages; while (scanf("%d %d", &tag, &stages) == 2) printf("%d\\n", last_copy(tag, stages)); }
""")
    subprocess.run(["g++", "-std=c++17", "-o", str(tmp_path / "rule"), str(tmp_path / "rule.cpp")], check=True)
    rng, asked, want = random.Random(1), [], []
    for stages, lanes in ((4, 1), (8, 8), (16, 8)):
        for n in range(0, 70):
            none = {i for i in range(n) if rng.random() < 0.2}           # pages with nothing to load
            stop = [rng.randint(0, n) for _ in range(lanes)]             # where each lane stopped
            tags, fills, loaded = [0] * stages, [0] * stages, [False] * stages
            for i in range(n):
                if i < stop[i % lanes]:
                    s = i % stages
                    tags[s], loaded[s], fills[s] = (-(i + 1) if i in none else i + 1), i not in none, fills[s] + 1
            asked += [(tag, stages) for tag in tags]
            # the f-th fill of a stage ends phase f - 1 of its barrier
            want += [(f - 1) % 2 if there else -1 for f, there in zip(fills, loaded)]
    out = subprocess.run([str(tmp_path / "rule")], input="\n".join(f"{t} {s}" for t, s in asked), capture_output=True, text=True, check=True)
    assert list(map(int, out.stdout.split())) == want
    kernel = text[text.index("decode_mma_kernel(const MmaParams"):text.index("// ---- merge the consumer warps")]
    issue, behind = kernel.split("__syncthreads();   // every page consumed")
    clear = "if (MASS && tid >= 32 && tid < 32 + kMmaStages) stage_tag[tid - 32] = 0;"
    assert issue.index(clear) < issue.index("__syncthreads();") and "never" not in issue      # nobody waits before the block has met
    assert re.search(r"for \(int s = 0; s < kMmaStages; \+\+s\) \{\s*const int phase = last_copy\(stage_tag\[s\], kMmaStages\);\s*"
                     r"if \(phase >= 0\) mbar_wait\(&full_bar\[s\], phase, &never\);", behind)
    assert behind.index("last_copy(") < behind.index("if (!MASS) return;")


def test_kernels_share_their_limits_of_shared_memory():
    """The limit belongs to the kernel: set per call, it is lowered under a launch of another thread.  One place sets it, and only raises it."""
    sources = [p for suffix in ("cu", "cuh") for p in CSRC.rglob(f"*.{suffix}")]
    assert [p.name for p in sources if "cudaFuncAttributeMaxDynamicSharedMemorySize" in p.read_text()] == ["ktk_host.cu"]
    assert sum("allow_shared(" in p.read_text() for p in sources) > 15


def test_nothing_is_thrown_where_kernels_limits_are_kept():
    text = (CSRC / "ktk_host.cu").read_text()
    body = text[text.index("cudaError_t raise_shared("):text.index("int sm_count()")]
    guarded = body[body.index("try {"):body.index("} catch (...) {")]
    assert all(x in guarded and x not in body.replace(guarded, "") for x in ("lock_guard", "most[kernel]", "cudaFuncSetAttribute"))


def test_the_package_needs_no_private_names_of_torch():
    names = ("_cuda_getDevice", "_cuda_getCurrentRawStream", "_cuda_cudaCachingAllocator_raw_alloc", "_cuda_cudaCachingAllocator_raw_delete")
    code = (f"import torch\nfor name in {names!r}:\n    if hasattr(torch._C, name):\n        delattr(torch._C, name)\n"
            "from kinetics_b200 import ops\nassert all(map(callable, (ops._current_device, ops._current_stream, ops._take, ops._give_back)))\n")
    subprocess.run([sys.executable, "-c", code], check=True, cwd=CSRC.parent.parent)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_workspaces_are_sized_from_python(dtype):
    i32, lib, code = (lambda n: (torch.int32, None, n)), _lib.load(), _lib.KTK_BF16 if dtype == torch.bfloat16 else _lib.KTK_F32
    for batch, new, most_new, heads, group, places, pages, window in ((1, 512, 512, 8, 4, 3000, 160, 64), (6, 3000, 700, 8, 8, 2600, 500, 0), (3, 7, 5, 2, 1, 90, -1, 0)):
        q, kv, mass = torch.Size((new, heads * group, 128)), torch.Size((999, 2, 16, heads, 128)), torch.Size((batch, heads, places))
        tables = (i32(pages if pages >= 0 else 77), i32(batch + 1), i32(batch), i32(batch + 1))
        need = ops._prefill_mass_plan(q, dtype, kv, dtype, mass, torch.float32, False, pages < 0, tables, most_new, window)[3]
        assert need > 0 and ops.prefill_mass_workspace_bytes(batch, new, most_new, heads, group, places, dtype, pages, window) == need
    shape = lambda n: _lib.Shape(n, 8, 4, 128, 16, code, 999)
    for batch, most, keep in ((1, 144, 2048), (48, 144, 2048), (2, 2048, 4096), (1, 40000, 4096)):
        assert ops.evict_workspace_bytes(batch, 8, most, keep) == lib.ktk_evict_workspace_bytes(shape(batch), most, keep)
    assert ops.evict_workspace_bytes(48, 8, 144, 2048) > 0 == ops.evict_workspace_bytes(1, 8, 144, 2048)
    with pytest.raises(TypeError, match="not supported"):
        ops.prefill_mass_workspace_bytes(1, 1, 1, 1, 1, 16, torch.float16)


@pytest.mark.parametrize("dtype", [0, 1])
def test_a_prompts_outputs_may_not_lie_on_its_queries(dtype):
    """The weights read the queries again.  Addresses are never dereferenced: what is not refused fails at the launch, which has no device."""
    lib, shape, one = _lib.load(), _lib.Shape(1, 2, 4, 128, 16, dtype, 8), 1 << 20
    bytes_ = 5 * 8 * 128 * (2 if dtype else 4)

    def call(o):
        return lib.ktk_prefill_attention_mass(one, 4096, 5, 5, 4096, 4096, 4096, 4096, None, 4, -1, 0, 0.1, _lib.Mass(4096, 4096, 64, 1, 1.0), o, 4096,
                                              1 << 20, shape, None, None)
    for o in (one, one + 256, one - 256, one + bytes_ - 16, one - bytes_ + 16):
        assert call(o) == -1 and b"q and o overlap" in lib.ktk_last_error()
    if not torch.cuda.is_available():
        assert call(one + bytes_) != -1 and call(one - bytes_) != -1


def test_a_slot_has_one_row():
    class Cfg:
        hidden_size, num_attention_heads, num_key_value_heads, head_dim, num_hidden_layers = 512, 4, 2, 128, 2

    kv = EvictingKVManager(Cfg, 3, 512, "meta", torch.bfloat16, keep=128)
    for slots in ([0, 0], [2, 1, 2], [3], [-1]):
        for call in (kv.begin_step, kv.prepare_step, lambda slots: kv._slots_of(torch.tensor(slots))):
            with pytest.raises(ValueError, match="different ones of 3"):
                call(slots)
    assert not kv._held.any() and not kv._seen.any()
    kv.begin_step(torch.tensor([2, 0]).tolist())
    assert kv._active == [2, 0]
