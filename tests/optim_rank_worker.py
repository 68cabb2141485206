"""One rank of tests/test_gpu_train_optim.py's exchange: steps of the flat buffer with 8-bit moments, weight decay and
clipping on the sum of all ranks' gradients.  gloo, on host copies of the gradients."""
import hashlib
import sys

import torch
import torch.distributed as dist


def buffer():
    from gsr import train
    spec = [("a", (7000, 3), 1e-2), ("b", (1,), 1e-3), ("c", (256,), 3e-3), ("d", (333, 45), 1e-4)]
    fp = train.FlatParams(spec, "cuda:0", moment_bits=8)
    g = torch.Generator().manual_seed(0)
    for name, shape, _ in spec:
        fp.load(name, torch.randn(shape, generator=g).to("cuda:0"))
    fp.set_weight_decay("a", 0.1)
    return fp


def gradient(fp, step, rank):
    g = torch.Generator().manual_seed(100 * step + rank)
    return torch.randn(fp.n, generator=g) * torch.exp(2 * torch.randn(fp.n, generator=g)) * 1e-3


def steps(world, exchanged, chunks):
    """A digest of the parameters, moments and clip coefficients after six steps.  exchanged(fp, step): the sum of the
    ranks' gradients."""
    from gsr import dp
    fp, said = buffer(), []
    for step in range(6):
        fp.grad.copy_(exchanged(fp, step))
        clip = fp.grad_norm(0.01, 1.0 / world)
        fp.begin_step(1.0 / world, clip)
        for lo, hi in dp.exchange_chunks(fp.n, chunks, 1, fp.align):
            fp.step_range(lo, hi)
        said.append(clip)
    h = hashlib.sha256()
    for t in (fp.flat.detach(), *fp.moments, torch.stack(said)):
        h.update(t.reshape(-1).view(torch.uint8).cpu().numpy().tobytes())
    return h.hexdigest()


def main(rank, world, port, to):
    dist.init_process_group("gloo", init_method=f"tcp://127.0.0.1:{port}", rank=rank, world_size=world)

    def exchanged(fp, step):
        x = gradient(fp, step, rank)
        dist.all_reduce(x)
        return x
    digest = steps(world, exchanged, 3 + rank)
    with open(f"{to}.{rank}", "w") as f:
        f.write(digest)
    dist.barrier()
    dist.destroy_process_group()


if __name__ == "__main__":
    main(int(sys.argv[1]), int(sys.argv[2]), int(sys.argv[3]), sys.argv[4])
