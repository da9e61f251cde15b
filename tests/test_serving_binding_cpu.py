"""The torch binding of the serving calls without a GPU: tensors that hold no
memory (their device and shape are all the checks look at) and what is refused
before anything is enqueued."""
import warnings

import pytest

torch = pytest.importorskip("torch")
from torch._subclasses.fake_tensor import FakeTensorMode  # noqa: E402

from xpose_b200 import serving as S  # noqa: E402

F16, F32, I32, I64, I8 = torch.float16, torch.float32, torch.int32, torch.int64, torch.int8
T, H, D = 4, 2, 64


def arguments(call):
    """The tensors of a call, by name and in order: shapes and types, and what is no tensor."""
    rows = lambda h=H: ((T, h, D), F16)  # noqa: E731
    pages = {n: ((8, H, 16, D), I8) for n in ("k_pages", "v_pages")} | {n: ((8, H, 16), F32) for n in ("k_scale", "v_scale")}
    attend = {"starts": ((2,), I32), "scratch": ((S.SCRATCH_BYTES,), torch.uint8), "lse": ((T, H), F32)}
    turn = {"positions": ((T,), I32), "turns": ((D // 2,), I64)}
    return {
        "rope_rows": {"out": rows(), "x": rows(), **turn},
        "kv_write": pages | {"k": rows(), "v": rows(), "slots": ((T,), I64), **turn},
        "kv_read": pages | {"k": rows(), "v": rows(), "slots": ((T,), I64)},
        "attention_packed": {"out": rows(), "q": rows(), "k": rows(), "v": rows(), **attend},
        "attention_paged": {"out": rows(), "q": rows(), **pages, "table": ((1, 8), I32), "kv_lens": ((1,), I32),
                            **attend, "q_most": 4},
    }[call]


def make(call, device=lambda name: "cuda:0"):
    with FakeTensorMode():
        return {n: torch.empty(a[0], dtype=a[1], device=device(n)) if isinstance(a, tuple) else a
                for n, a in arguments(call).items()}


CALLS = ["rope_rows", "kv_write", "kv_read", "attention_packed", "attention_paged"]


def refused(call, args, *words):
    with warnings.catch_warnings():
        warnings.simplefilter("ignore")
        with pytest.raises(S.XpError) as e:
            getattr(S, call)(**args)
    assert e.value.name == "XP_ERR_INVALID", e.value
    for w in words:
        assert w in str(e.value), e.value


@pytest.mark.parametrize("call,odd", [(c, n) for c in CALLS for n, a in arguments(c).items() if isinstance(a, tuple)])
def test_one_tensor_on_another_device_is_refused(call, odd):
    refused(call, make(call, lambda name: "cuda:1" if name == odd else "cuda:0"), "device 0", "device 1")


@pytest.mark.parametrize("call,odd", [(c, n) for c in CALLS for n, a in arguments(c).items() if isinstance(a, tuple)])
def test_a_tensor_on_the_host_is_refused(call, odd):
    refused(call, make(call, lambda name: "cpu" if name == odd else "cuda:0"), f"'{odd}'", "CUDA")


@pytest.mark.parametrize("call,name", [("rope_rows", "magnitude"), ("kv_write", "magnitude"),
                                       ("attention_packed", "scale"), ("attention_paged", "scale")])
@pytest.mark.parametrize("value", ["one", None, [1.0]])
def test_what_is_no_number_is_refused_before_anything_is_enqueued(call, name, value):
    refused(call, make(call) | {name: value}, f"'{name}'", "number")


@pytest.mark.parametrize("call,name", [("attention_packed", "window"), ("attention_paged", "window"),
                                       ("attention_paged", "q_most")])
@pytest.mark.parametrize("value", ["one", None, 1.5, -1, 1 << 31])
def test_what_is_no_count_is_refused(call, name, value):
    refused(call, make(call) | {name: value}, f"'{name}'", "whole number")


def test_a_direction_without_truth_value_is_refused():
    refused("rope_rows", make("rope_rows") | {"inverse": torch.ones(2)}, "'inverse'")
