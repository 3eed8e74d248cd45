"""Which tensors the Python launchers of the 4-bit cache and log probabilities take: all on one GPU, the stream's
(checked before the library is called; no GPU needed)."""
import pytest
import torch


class Elsewhere:
    """Stands for a tensor of GPU 1."""
    device = "cuda:1"

    def __init__(self, gpu=1):
        self.gpu = gpu

    def get_device(self):
        return self.gpu

    def data_ptr(self):
        return 1 << 20


class Stream:
    cuda_stream, device_index = 0x5000, 0


# every tensor argument of every launcher, as numbers: addresses pass unlooked at
CALLS = [("launch_qkv_bias_rope_kv4_append", 11, (1,)), ("launch_kv4_unpack", 4, (0, 1)),
         ("launch_attention_gqa_flash_decode_kv4", 7, ()), ("launch_attention_gqa_prefill_kv4", 6, (1,)),
         ("launch_kv4_evict", 10, (8, 1, 1)), ("launch_token_logprobs", 7, (1,))]
NAMED = {"launch_attention_gqa_flash_decode_kv4": ("out_q8", "out_scale", "out_sum8", "key_weights_in", "key_weights_out"),
         "launch_attention_gqa_prefill_kv4": ("key_weights_in", "key_weights_out", "row_lse")}
EACH = [(name, n, rest, which) for name, n, rest in CALLS for which in (*range(n), *NAMED.get(name, ()))]


def _call(name, n, rest, given, stream):
    """The call with addresses that nothing takes (odd ones, which the library would refuse) but for `given`."""
    import qe_amd
    args = [0xFFF1 + 0x10000 * i for i in range(n)]
    named = {}
    for which, tensor in given.items():
        if isinstance(which, int):
            args[which] = tensor
        else:
            named[which] = tensor
    return getattr(qe_amd, name)(*args, *rest, stream=stream, **named)


@pytest.mark.parametrize("stream", [None, 0x5000, Stream()], ids=["current", "handle", "stream"])
@pytest.mark.parametrize("name,n,rest,which", EACH)
def test_one_tensor_in_host_memory(name, n, rest, which, stream):
    with pytest.raises(RuntimeError, match="must be on a GPU"):
        _call(name, n, rest, {which: torch.zeros(4096, dtype=torch.uint8)}, stream)


@pytest.mark.parametrize("name,n,rest,which", EACH)
def test_one_tensor_of_another_gpu(name, n, rest, which):
    with pytest.raises(RuntimeError, match="cuda:1"):
        _call(name, n, rest, {which: Elsewhere()}, Stream())
    other = 0 if which != 0 else 1
    with pytest.raises(RuntimeError, match="on one GPU"):
        _call(name, n, rest, {other: Elsewhere(0), which: Elsewhere()}, 0x5000)


@pytest.mark.parametrize("name,n,rest", CALLS)
def test_tensors_of_one_gpu_reach_the_library(name, n, rest):
    """The library's own refusal of the odd addresses, or of what is missing, says that it was called."""
    for stream in (0x5000, Stream()):
        with pytest.raises(RuntimeError, match="failed"):
            _call(name, n, rest, {0: Elsewhere(0)}, stream)
