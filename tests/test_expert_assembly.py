"""What the compiled code of the expert kernels has to keep, read from its assembly (device side only, no GPU needed).

The compiler inserts the wait states that the hardware asks for between instructions, but does not look into inline
assembly: what is written there has to hold whatever the compiler puts in front of it and behind it."""
import concurrent.futures
import os
import re
import subprocess

import pytest

from brainpylib_amd import build

SOURCES = ["expert_matmul.hip", "expert_route.hip"]


def _assembly(src, out_dir):
  out = os.path.join(out_dir, src[:-4] + ".s")
  flags = [f for f in build.HIP_FLAGS if f not in ("-fPIC", "-Wall")]
  cmd = [build.HIPCC] + flags + ["-S", "--cuda-device-only", "-I" + os.path.join(os.path.dirname(build.CSRC), "..", "include"),
                                 os.path.join(build.CSRC, src), "-o", out]
  r = subprocess.run(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
  assert r.returncode == 0, r.stdout[-2000:]
  with open(out) as f:
    return f.read()


@pytest.fixture(scope="module")
def assembly(tmp_path_factory):
  if not os.path.exists(build.HIPCC):
    pytest.skip("no hipcc")
  out_dir = str(tmp_path_factory.mktemp("asm"))
  with concurrent.futures.ThreadPoolExecutor(max_workers=len(SOURCES)) as ex:
    return dict(zip(SOURCES, ex.map(lambda s: _assembly(s, out_dir), SOURCES)))


def registers(operand):
  """{(kind, number)} of an operand, modifiers left aside."""
  found = set()
  for word in operand.split():
    m = re.fullmatch(r"([vsa])(?:(\d+)|\[(\d+):(\d+)\])", word)
    if m:
      first = int(m.group(2) or m.group(3))
      found |= {(m.group(1), i) for i in range(first, int(m.group(4) or first) + 1)}
  return found


def instructions(text):
  """[(line, name, operands, whether it stands in inline assembly)]; labels are left out."""
  out, inline = [], False
  for number, line in enumerate(text.splitlines(), 1):
    if "#ASMSTART" in line or "#ASMEND" in line:
      inline = "#ASMSTART" in line
      continue
    line = line.split(";")[0].strip()
    if not line or line.startswith(".") or line.endswith(":"):
      continue
    name, _, rest = line.partition(" ")
    name, _, tab = name.partition("\t")
    out.append((number, name, [o.strip() for o in (tab + " " + rest).split(",")], inline))
  return out


def wait_states(name, operands):
  return int(operands[0], 0) + 1 if name == "s_nop" else 1


def overwritten_store_data(code):
  """Stores of more than 64 bits whose data a vector instruction overwrites less than two wait states later."""
  found = []
  for k, (line, name, operands, _) in enumerate(code):
    if not re.match(r"(global|flat|buffer|scratch)_store_dwordx[34]", name):
      continue
    data, passed = registers(operands[0 if name.startswith("buffer") else 1]), 0
    for line2, name2, operands2, _ in code[k + 1:k + 3]:
      if passed >= 2:
        break
      if name2.startswith("v_") and registers(operands2[0]) & data:
        found.append("%d: %s %s, %d: %s %s" % (line, name, operands, line2, name2, operands2))
      passed += wait_states(name2, operands2)
  return found


def early_scalar_reads(code):
  """Memory instructions in inline assembly that read a scalar register less than five wait states after a vector
  instruction has written it."""
  found = []
  for k, (line, name, operands, inline) in enumerate(code):
    if not inline or not re.match(r"(global|flat|buffer|scratch)_", name):
      continue
    read, passed = {r for o in operands for r in registers(o) if r[0] == "s"}, 0
    for line2, name2, operands2, _ in reversed(code[max(k - 5, 0):k]):
      if passed >= 5:
        break
      # (an instruction that carries writes its second operand too)
      written = operands2[:2 if "_co_" in name2 else 1]
      if name2.startswith("v_") and read & {r for o in written for r in registers(o)}:
        found.append("%d: %s %s, %d: %s %s" % (line, name, operands, line2, name2, operands2))
      passed += wait_states(name2, operands2)
  return found


def test_the_checks_find_what_they_look_for():
  store = "\tglobal_store_dwordx4 v[0:1], v[4:7], off nt\n"
  write = "\tv_lshl_add_u64 v[6:7], v[0:1], 0, s[2:3]\n"
  for between, found in (("", 1), ("\ts_nop 0\n", 1), ("\ts_nop 1\n", 0), ("\ts_nop 0\n\ts_nop 0\n", 0), ("\tv_mov_b32_e32 v9, v8\n", 1)):
    assert len(overwritten_store_data(instructions(store + between + write))) == found, between
  assert not overwritten_store_data(instructions(store + "\tv_mov_b32_e32 v8, v7\n"))
  write, load = "\tv_readfirstlane_b32 s4, v1\n", "\t;#ASMSTART\n\ts_mov_b32 m0, s9\n\ts_nop 0\n\tglobal_load_lds_dwordx4 v2, s[4:5] nt\n\t;#ASMEND\n"
  assert len(early_scalar_reads(instructions(write + load))) == 1
  assert len(early_scalar_reads(instructions(write + "\ts_nop 1\n" + load))) == 1
  assert not early_scalar_reads(instructions(write + "\ts_nop 2\n" + load))


def test_data_of_wide_stores_is_left_alone_until_it_is_read(assembly):
  # gfx950 reads the data of a store of more than 64 bits after it has issued the next instruction: a vector instruction may
  # overwrite it two wait states later at the earliest
  for source, text in assembly.items():
    code = instructions(text)
    assert sum(bool(re.match(r"global_store_dwordx4", i[1])) for i in code) > 10, source
    assert not overwritten_store_data(code), source


def test_scalar_addresses_are_written_in_time(assembly):
  code = instructions(assembly["expert_matmul.hip"])
  assert sum(i[3] and i[1].startswith("global_load_lds") for i in code) > 100
  assert not early_scalar_reads(code)


def test_what_the_loads_to_lds_are_told_is_nothing_elses(assembly):
  # (m0 is reserved: the compiler takes no note of an assembly statement that writes it, and must have no use of its own for it)
  for source, text in assembly.items():
    assert not [i for i in instructions(text) if not i[3] and any("m0" in o.split() for o in i[2])], source


# Vector registers that the kernels of the largest tiles spill, at most: (part of the mangled name, registers).  The main loop has
# none of it, the way of the results out has.
SPILLS = [(r"14product_kernelI.*Lb1ENS_5ShapeILj256ELj256ELj2ELj2E.*ES2_EEv", 72),
          (r"14product_kernelI.*Lb0ENS_5ShapeILj256ELj256ELj2ELj2E.*ES2_EEv", 116),
          (r"14product_kernelI.*Lb[01]ENS_5ShapeILj256ELj256ELj2ELj4E.*ES2_EEv", 24),
          (r"15gradient_kernelI.*NS_5ShapeILj256ELj256ELj2ELj2E", 60)]


def kernels(text):
  """[(mangled name, bytes of scratch memory a lane, vector registers spilled)]"""
  pattern = r"\.name:\s+(\S+)\n(?:.*\n)*?\s+\.private_segment_fixed_size:\s+(\d+)\n(?:.*\n)*?\s+\.vgpr_spill_count:\s+(\d+)"
  return [(n, int(b), int(r)) for n, b, r in re.findall(pattern, text[text.index("amdhsa.kernels"):])]


def test_only_the_largest_tiles_spill(assembly):
  seen, over = 0, []
  for text in assembly.values():
    for name, scratch, spilled in kernels(text):
      most = max([n for part, n in SPILLS if re.search(part, name)], default=0)
      seen += 1
      if spilled > most or (most == 0 and scratch):
        over.append("%s: %d registers, %d bytes a lane" % (name, spilled, scratch))
  assert seen > 100 and not over, over


def test_the_main_loop_of_the_largest_tiles_does_not_spill(assembly):
  # somewhere a stage's 64 matrix instructions (four steps of 4 x 4; 32 of the waves that take 128 x 64) follow each other with no
  # spilled register stored or fetched between them
  text, seen = assembly["expert_matmul.hip"], 0
  for name, scratch, _ in kernels(text):
    if not scratch:
      continue
    begin = text.index("\n%s:" % name)
    code = instructions(text[begin:text.index("s_endpgm", begin)])
    runs = "".join("m" if i[1].startswith("v_mfma") else "s" if i[1].startswith("scratch_") else "" for i in code).split("s")
    assert max(map(len, runs)) >= (32 if "ILj256ELj256ELj2ELj4E" in name else 64), name
    seen += 1
  assert seen >= 6
