"""CPU tests: tensors that a KV cache cannot be made of, whatever the size of their elements, and caches in host memory."""
import pytest
import torch


def tensors():
    return torch.zeros((3, 2, 16, 64), dtype=torch.int8), torch.zeros((3, 2, 16, 64), dtype=torch.int8), torch.zeros((3, 2)), torch.zeros((3, 2))


@pytest.mark.parametrize("at,dtype", [(0, torch.uint8), (1, torch.bool), (0, torch.float8_e4m3fn), (2, torch.int32), (3, torch.uint32)])
def test_other_types_of_the_same_size(w4a8, at, dtype):
    t = list(tensors())
    t[at] = t[at].to(dtype)
    with pytest.raises(ValueError, match="int8 codes and fp32 scales"):
        w4a8.KVCache.of(*t)


def test_tensors_on_several_devices(w4a8):
    k, v, ks, vs = tensors()
    with pytest.raises(ValueError, match="one device"):
        w4a8.KVCache.of(k, v, ks, vs.to("meta"))


def test_launches_refuse_a_cache_in_host_memory(w4a8):
    c = w4a8.KVCache.of(*tensors())
    x, i = torch.zeros((1, 128)), torch.zeros(4, dtype=torch.int32)
    for call in (lambda: w4a8.launch_kv_append_q8(x, x, 128, i, 1, c), lambda: w4a8.launch_kv_read_q8(c, i, 1, i, i, 1, 1, x, x, 128),
                 lambda: w4a8.launch_attention_q8(x, 128, c, i, 1, i, i, 1, 1, 2, x, 128, 0.1, "fp32", torch.zeros(1 << 20, dtype=torch.uint8))):
        with pytest.raises(ValueError, match="not on a GPU"):
            call()
