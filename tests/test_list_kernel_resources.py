"""What the compiler says about the kernels over a row and a list of tokens (registers, scratch, LDS), on the
CPU: compiled for gfx950 with the library's own flags, those of the single source included."""
import functools
import os
import re
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@functools.lru_cache(maxsize=None)
def _resources(source):
    """{mangled kernel name: {"VGPRs": n, "VGPRs Spill": n, "ScratchSize": n, "LDS Size": n}}"""
    from openrlhf_amd.csrc import build as b

    cmd = [b.find_hipcc(), *b.HIPCC_FLAGS, *b.SOURCE_FLAGS.get(source, []), "-I", os.path.join(ROOT, "include"), "--cuda-device-only",
           "-c", os.path.join(b.CSRC, source), "-o", os.devnull, "-Rpass-analysis=kernel-resource-usage"]
    out = subprocess.run(cmd, capture_output=True, text=True)
    assert out.returncode == 0, out.stderr[-2000:]
    kernels, name = {}, None
    for line in out.stderr.splitlines():
        m = re.search(r"remark:\s+Function Name: (\S+)", line)
        if m:
            name = m.group(1)
            kernels[name] = {}
            continue
        m = re.search(r"remark:\s+(VGPRs Spill|VGPRs|ScratchSize|LDS Size)(?: \[[^]]*\])?: (\d+)", line)
        if m and name:
            kernels[name][m.group(1)] = int(m.group(2))
    return kernels


def test_candidate_keys_lie_on_16_bytes():
    """The ranking reads the candidates two keys at a time with 16-byte LDS loads. In the forward kernel they
    lie in the dynamic LDS, which begins where the static LDS ends."""
    kernels = {k: v for k, v in _resources("top_logprobs.hip").items() if "top_logprobs_fwd_kernel" in k}
    assert len(kernels) == 9, sorted(kernels)
    for k, v in kernels.items():
        assert v["LDS Size"] > 0 and v["LDS Size"] % 16 == 0, (k, v)


def test_one_pass_distillation_fits_the_lds_of_a_cu(lib):
    """Static LDS as compiled, two maps of the longest row (a bit per element, whole 16-byte words) and the six
    parked 16-byte chunks of 512 lanes in the 160 KiB of a CU."""
    from openrlhf_amd import _lib

    longest = max(lib.orlhf_distill_kl_fwd_bwd_max_vocab(t) for t in (_lib.F32, _lib.BF16, _lib.F16))
    maps, parked = 2 * ((longest + 127) // 128 * 16), 6 * 512 * 16
    kernels = {k: v for k, v in _resources("distill_fused.hip").items() if "distill_one_pass_kernel" in k}
    assert len(kernels) == 6, sorted(kernels)
    for k, v in kernels.items():
        assert v["LDS Size"] + maps + parked <= 160 * 1024, (k, v)


def test_one_pass_distillation_does_not_spill():
    """A body holds a whole vocabulary row in its registers: nothing else of the kernel may push any of it to
    scratch memory, in none of the three types, short rows or long."""
    kernels = {k: v for k, v in _resources("distill_fused.hip").items() if "distill_one_pass_kernel" in k}
    assert len(kernels) == 6, sorted(kernels)
    for k, v in kernels.items():
        assert v["VGPRs Spill"] == 0 and v["ScratchSize"] == 0, (k, v)
