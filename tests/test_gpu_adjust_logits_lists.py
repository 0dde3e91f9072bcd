"""adjust_logits: long lists of biases that name the same tokens again and again, and what a call's indexes hold."""
import numpy as np
import pytest

from test_gpu_adjust_logits import Case, _run

pytestmark = pytest.mark.gpu

LISTS = {
    "one": lambda g: np.full(1024, 5),
    "two": lambda g: np.where(np.arange(1024) % 3 == 0, 70000, 4),
    "pairs": lambda g: np.repeat(np.arange(512) * 8, 2),
    "padded": lambda g: np.concatenate([g.choice(73448, 40, replace=False), np.full(984, 73447)]),
    "mixed": lambda g: g.integers(-1, 300, 1024),
    "three": lambda g: np.array([9, 9, 9]),
}


@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("name", list(LISTS))
@pytest.mark.parametrize("L", [0, 6000, 9000])
def test_lists_that_repeat(gpu, set_option, dtype, name, L):
    """Added up in the order of the list, in 32 bits."""
    from cpm.cu_amd import synth
    set_option("dtype", dtype)
    ids = LISTS[name](synth.rng(80, 1))
    case = Case(gpu, 80, n=2, V=73448, nb=len(ids), L=L, mask=L > 0, dtype=dtype)
    case.bias_ids[0] = ids
    case.bias_ids[1] = ids[::-1]
    out, best = _run(case)
    case.check(out, best)


def test_a_list_of_one_token_takes_no_longer(gpu):
    """One slice has all of the list: it is added up in one pass, so the call takes a few times what a list of other tokens takes at most (a pass for each entry: hundreds)."""
    torch = gpu
    from cpm.cu_amd import ops
    z = torch.randn((4, 73448), device="cuda").half()
    values = torch.randn((4, 1024), device="cuda")
    lists = [torch.arange(1024, dtype=torch.int32, device="cuda").mul_(70).repeat(4, 1), torch.full((4, 1024), 77, dtype=torch.int32, device="cuda")]
    times = [[], []]
    for _ in range(5):
        for i, ids in enumerate(lists):
            begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            ops.adjust_logits(z, bias_ids=ids, bias_values=values)
            begin.record()
            for _ in range(5):
                ops.adjust_logits(z, bias_ids=ids, bias_values=values)
            end.record()
            end.synchronize()
            times[i].append(begin.elapsed_time(end))
    assert min(times[1]) < 20 * min(times[0]), times


@pytest.mark.parametrize("n", [0, 1, 2, 7, 512])
def test_indexes_hold_nothing_else(gpu, n):
    """A kept tensor of indexes keeps no workspace, and a saved one writes none."""
    torch = gpu
    from cpm.cu_amd import ops
    z = torch.randn((n, 9001), device="cuda").half()
    _, ids = ops.adjust_logits(z)
    assert ids.storage_offset() == 0 and ids.untyped_storage().nbytes() == 4 * n
    assert torch.equal(ids.long(), z.float().argmax(1))
