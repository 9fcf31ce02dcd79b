"""Graph captures beside a process group's watchdog thread."""
import socket

import torch.distributed as dist

from sequoia_amd.Engine.ts_linear import capture_mode


def test_captures_watch_their_own_thread_alone_while_a_process_group_lives():
    assert not dist.is_initialized() and capture_mode() == "global"
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    dist.init_process_group("gloo", init_method=f"tcp://127.0.0.1:{port}", rank=0, world_size=1)
    try:
        assert capture_mode() == "thread_local"
    finally:
        dist.destroy_process_group()
    assert capture_mode() == "global"
