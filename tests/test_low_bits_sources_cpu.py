"""Order of memory in the kernels of few bits, as far as their text shows it. Such a kernel is launched while the one before it still runs:
what another kernel writes must not be read by loads that are only right for memory that nobody writes while the kernel runs."""
import os
import re

import nanoinfer_b200.csrc as csrc

HERE = os.path.dirname(csrc.__file__)
# a step's inputs and a model's parameters: what may be read ahead of the wait and past the coherent loads
INPUTS = {"ctx_lens", "q_start", "block_table", "bt", "bias"}
PARAMETERS_OF_UNPACK = {"w", "scales"}          # codes and scales of 4-bit weights


def code(name):
    with open(os.path.join(HERE, name)) as f:
        return re.sub(r"//[^\n]*", "", f.read())


def kernels(text):
    """(name, parameters, body) of every kernel."""
    for m in re.finditer(r"__global__ void __launch_bounds__\([^\n]*\)\s*\n(\w+)\(", text):
        depth, at = 1, m.end()
        while depth:
            depth += {"(": 1, ")": -1}.get(text[at], 0)
            at += 1
        begin = text.index("{", at)
        depth, end = 1, begin + 1
        while depth:
            depth += {"{": 1, "}": -1}.get(text[end], 0)
            end += 1
        yield m.group(1), text[m.end():at], text[begin:end]


def test_results_of_other_kernels_are_read_coherently():
    seen = set()
    for name in ("attention_int8.cu", "cache_int8.cu", "gemm_int4.cu"):
        text = code(name)
        for kernel, params, body in kernels(text):
            seen.add(kernel)
            allowed = INPUTS | (PARAMETERS_OF_UNPACK if kernel == "unpack_int4_kernel" else set())
            bare = set(re.findall(r"const [\w ]+\* __restrict__ (\w+)", params))
            assert bare <= allowed, (name, kernel, bare - allowed)
            for source in re.findall(r"__ldg\((?:reinterpret_cast<[^>]*>\()?(?:a\.)?(\w+)", body):
                assert source in allowed, (name, kernel, source)
    assert {"attention_int8_mma_kernel", "attention_int8_any_kernel", "merge_int8_kernel", "append_int8_kernel", "unpack_int8_kernel", "gather_int8_kernel",
            "prepare_f16_kernel", "gemm_int4_kernel", "unpack_int4_kernel"} <= seen


def test_every_kernel_waits_before_it_reads_rows_and_pools_and_before_it_writes():
    """What a kernel behind the wait of the one before it sees is not what the kernels before both have written unless it waits itself."""
    (append,) = [body for name, _, body in kernels(code("cache_int8.cu")) if name == "append_int8_kernel"]
    before, _, behind = append.partition("\n    pdl_wait();\n")         # (the CTAs of keys and values: a statement of its own, under no condition)
    assert behind, "no unconditional wait"
    for touched in ("k_codes", "v_codes", "k_rows", "v_rows", "k_scales", "v_scales"):
        assert touched not in before and touched in behind, touched


def test_no_scale_is_sent_for_ahead_of_the_wait():
    """Scales of several pages share 32 bytes: one that is fetched early would bring in the one that the append before is writing."""
    (body,) = [body for name, _, body in kernels(code("attention_int8.cu")) if name == "attention_int8_mma_kernel"]
    early = body[body.index("a.early"):body.index("pdl_wait();")]
    calls = re.findall(r"\bsend\w*\([^;]*;", early)
    assert calls and all(c.startswith("send(") and c.endswith("std::false_type{});") for c in calls)        # (the codes alone)
    assert re.search(r"auto send = \[&\]\(int chunk, int stage, auto with_scales\)", body)
