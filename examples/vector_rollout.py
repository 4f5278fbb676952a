"""A rollout loop through the batched user surface (agarcl_amd/vector_env.py: AgarioVectorEnv): N arenas, a random policy on the device,
T steps collected into a rollout buffer -- the shape of a PPO / IMPALA actor -- with nothing inside the loop that waits for the GPU.

    python examples/vector_rollout.py [--envs 4096] [--steps 256] [--obs grid|ram|screen|none] [--difficulty normal] [--mode 6] [--sub-batches auto|k [--halves]]
    python examples/vector_rollout.py --learn [--updates 3]

--sub-batches k: the arenas as k independent ranges on HIP streams of their own (a range never waits for the slowest arena of another, one
range's observation kernel runs under another's step).  The default, "auto", is what AgarioVectorEnv picks: ONE range for the full-batch
step() (which orders every range against the caller's stream every step: measured slower with ranges, scripts/gpu_vec_pipe_ab.py), and with
--halves agarcl_amd/vec_env.py default_sub_batches: 4 where the general engine handles most arena-steps -- bots, several agents, modes 5 / 6
(try --mode 6 --halves) --, 1 for quiet batches such as the default mode 0.
--learn: a policy with a memory instead of the random one, and `--updates` policy-gradient updates on the rollouts it collects, through agarcl_amd/learn.py:
recurrence_step and sample_actions between the steps, advantages, gated_recurrence and policy_loss on the rollout (observation "ram").
--halves: double-buffered sampling through recv(j) / send(actions_j, j) -- the policy works on range j's observations while the other ranges step.

Prints env-steps per second of the whole loop (engine step + observation + Python), which is what a learner sees; `bench.py` times the
engine alone."""
import argparse, os, sys, time
sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))   # (run from a checkout: the package is in-tree)
import torch
from agarcl_amd.vector_env import AgarioVectorEnv

ap = argparse.ArgumentParser()
ap.add_argument("--envs", type=int, default=4096); ap.add_argument("--steps", type=int, default=256)
ap.add_argument("--obs", default="ram"); ap.add_argument("--difficulty", default="normal"); ap.add_argument("--number-steps", type=int, default=500)
ap.add_argument("--bare", action="store_true", help="time venv.step alone: one fixed action batch, no rollout buffer")
ap.add_argument("--sub-batches", default="auto", type=lambda v: v if v == "auto" else int(v)); ap.add_argument("--halves", action="store_true", help="recv / send per sub-batch instead of full-batch step()")
ap.add_argument("--mode", type=int, default=0)
ap.add_argument("--learn", action="store_true", help="collect with a recurrent policy and update it"); ap.add_argument("--updates", type=int, default=3)
a = ap.parse_args()
venv = AgarioVectorEnv(a.envs, obs_type=a.obs, difficulty=a.difficulty, number_steps=a.number_steps, env_type=0, sub_batches=a.sub_batches, halves=a.halves, mode=a.mode,
                       **({"num_viruses": 25} if a.mode else {}))
dev = venv.device
obs, _ = venv.reset(seed=1)
g = torch.Generator(device=dev); g.manual_seed(0)
buf_obs = None if obs is None else torch.empty((a.steps,) + tuple(obs.shape), dtype=obs.dtype, device=dev)
buf_rew = torch.empty((a.steps, a.envs), dtype=torch.float32, device=dev)
buf_done = torch.empty((a.steps, a.envs), dtype=torch.bool, device=dev)
def policy():   # uniform moves, action kind ~ U{none, feed, split}
    return torch.rand((a.envs, 2), generator=g, device=dev) * 2 - 1, torch.randint(0, 3, (a.envs,), generator=g, device=dev, dtype=torch.int32)
if a.learn:
    from agarcl_amd import learn
    if a.obs != "ram": sys.exit("--learn works on the ram observation")
    T, N, D, C = a.steps, a.envs, obs.shape[-1], 128
    w = {k: (torch.randn(shape, generator=g, device=dev) / shape[0] ** 0.5).requires_grad_() for k, shape in
         dict(x=(D, C), gate=(D, C), kind=(C, 3), mean=(C, 2), value=(C, 1)).items()}
    w["log_std"] = torch.full((2,), -0.5, device=dev, requires_grad=True)
    opt = torch.optim.Adam(w.values(), lr=3e-4)
    see = lambda o: torch.tanh(o * 0.01)
    memory, ended = torch.zeros(N, C, device=dev), torch.ones(N, dtype=torch.bool, device=dev)
    new = lambda *shape, dtype=torch.float32: torch.empty((T, N) + shape, dtype=dtype, device=dev)
    ob, reset, kind, raw, log_prob, value, reward, term, trunc = (new(D), new(dtype=torch.bool), new(dtype=torch.int32), new(2), new(), new(), new(), new(dtype=torch.bool),
                                                                  new(dtype=torch.bool))
    for update in range(a.updates):
        torch.cuda.synchronize(); t0 = time.perf_counter(); start = memory
        with torch.no_grad():
            gumbel, normal = -torch.log(torch.empty((T, N, 3), device=dev).exponential_(generator=g)), torch.randn((T, N, 2), generator=g, device=dev)   # one launch each for the whole rollout
            for t in range(T):
                ob[t].copy_(see(obs)); reset[t].copy_(ended)
                h, memory = learn.recurrence_step(ob[t] @ w["x"], ob[t] @ w["gate"], memory, reset[t])
                act = learn.sample_actions(h @ w["kind"], h @ w["mean"], w["log_std"], gumbel=gumbel[t], normal=normal[t])
                obs, rew, te, tr, info = venv.step(act)
                for buf, v in ((kind, act.kind), (raw, act.raw), (log_prob, act.log_prob), (value, (h @ w["value"])[:, 0]), (reward, rew), (term, te), (trunc, tr)): buf[t].copy_(v)
                ended = info["ended"]
            o = see(obs)      # the value behind the last step: of the state the next one will have
            h, _ = learn.recurrence_step(o @ w["x"], o @ w["gate"], memory, ended)
            adv, ret = learn.advantages(reward, value, (h @ w["value"])[:, 0], term, trunc)
            adv = (adv - adv.mean()) / (adv.std() + 1e-8)
        torch.cuda.synchronize(); t1 = time.perf_counter()
        h, _ = learn.gated_recurrence(ob @ w["x"], ob @ w["gate"], start, reset)
        out = learn.policy_loss(h @ w["kind"], kind, log_prob, adv, h @ w["mean"], w["log_std"], raw, kl_coef=0.01, entropy_coef=0.01)
        loss = out.loss + 0.5 * ((h @ w["value"])[..., 0] - ret).square().mean()
        opt.zero_grad(); loss.backward(); opt.step()
        torch.cuda.synchronize(); t2 = time.perf_counter()
        print("update %d: %d envs x %d steps collected in %.1f ms (%.3g env-steps/s), learned from in %.1f ms; loss %.4f kl %.2e entropy %.3f clipped %.3f, mean reward %.3f"
              % (update, N, T, (t1 - t0) * 1e3, N * T / (t1 - t0), (t2 - t1) * 1e3, loss.item(), out.kl.item(), out.entropy.item(), out.clipped.item(), reward.mean().item()))
    venv.close(); sys.exit(0)
for _ in range(8): venv.step(policy())                      # warm-up
if a.bare:
    act = policy(); torch.cuda.synchronize(); t0 = time.perf_counter()
    for t in range(a.steps): venv.step(act)
    torch.cuda.synchronize(); dt = time.perf_counter() - t0
    print("%d envs x %d steps, obs=%s, step() alone: %.3g env-steps/s (%.1f us per vector step)" % (a.envs, a.steps, a.obs, a.envs * a.steps / dt, dt / a.steps * 1e6))
    venv.close(); sys.exit(0)
if a.halves:   # every range on its own: range j's policy output is computed from range j's observation while the other ranges step
    k = venv.sub_batches
    def policy_j(n):
        return torch.rand((n, 2), generator=g, device=dev) * 2 - 1, torch.randint(0, 3, (n,), generator=g, device=dev, dtype=torch.int32)
    torch.cuda.synchronize(); t0 = time.perf_counter()
    ended = [torch.zeros((), dtype=torch.int64, device=dev) for _ in range(k)]
    for t in range(a.steps):
        for j in range(k):
            with torch.cuda.stream(venv.stream(j)):                   # range j's copies and policy on range j's own stream: no cross-stream ordering
                obs_j, rew_j, term_j, trunc_j, info_j = venv.recv(j)
                lo, cnt = venv.ranges[j]
                if buf_obs is not None: buf_obs[t, lo:lo + cnt].copy_(obs_j)
                buf_rew[t, lo:lo + cnt].copy_(rew_j); buf_done[t, lo:lo + cnt].copy_(term_j)
                ended[j] += info_j["ended"].sum()
                venv.send(policy_j(cnt), j)
    torch.cuda.synchronize(); dt = time.perf_counter() - t0
    print("%d envs x %d steps as %d ranges (recv / send halves), obs=%s: %.3g env-steps/s (%.1f us per vector step); %d episodes ended"
          % (a.envs, a.steps, k, a.obs, a.envs * a.steps / dt, dt / a.steps * 1e6, sum(int(e.item()) for e in ended)))
    venv.close(); sys.exit(0)
torch.cuda.synchronize(); t0 = time.perf_counter()
episodes = torch.zeros((), dtype=torch.int64, device=dev); ret_sum = torch.zeros((), dtype=torch.float32, device=dev)
for t in range(a.steps):
    obs, rew, term, trunc, info = venv.step(policy())
    if buf_obs is not None: buf_obs[t].copy_(obs)           # (the env rewrites its tensors in place: a rollout buffer copies them)
    buf_rew[t].copy_(rew); buf_done[t].copy_(term)
    episodes += info["ended"].sum(); ret_sum += (info["final_return"] * info["ended"]).sum()
torch.cuda.synchronize(); dt = time.perf_counter() - t0
n = int(episodes.item())
print("%d envs x %d steps, obs=%s: %.3g env-steps/s through AgarioVectorEnv.step (%.1f us per vector step); %d episodes ended, mean return %.1f"
      % (a.envs, a.steps, a.obs, a.envs * a.steps / dt, dt / a.steps * 1e6, n, float(ret_sum.item()) / max(n, 1)))
venv.close()
