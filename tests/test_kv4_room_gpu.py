"""How many blocks of attention over a 4-bit cache a GPU is taken to hold: what its registers and shared memory allow, form by form."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_each_form_is_asked_for_itself():
    from llm_singularity_b200 import kernels as ops
    ops.prepare(["attention_kv4", "attention_kv4_f32"])
    rooms = {}
    for lib, most in (("attention_kv4", 128), ("attention_kv4_f32", 0)):
        for hd in range(32, 257, 32):
            for eights in (1, 2) if hd <= most else (1,):
                for spread in (0, 1):
                    rooms[lib, hd, eights, spread] = ops._kv4_room(lib, hd, eights, spread, torch.device("cuda:0"))
    sms = ops.num_sms(torch.device("cuda:0"))
    # (every kernel's launch bounds ask for two blocks an SM; more where registers and shared memory have room)
    assert all(n % sms == 0 and 2 * sms <= n <= 16 * sms for n in rooms.values()), rooms
    assert all(n <= rooms[lib, hd, eights, 0] for (lib, hd, eights, spread), n in rooms.items()), rooms
    assert ops._kv4_room("attention_kv4", 64, 3, 1, torch.device("cuda:0")) == 0
